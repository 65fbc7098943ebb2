// sorted.hip -- rows sorted by expert and back (coli_hip_dispatch_dev,
// coli_hip_combine_dev, coli_hip_combine_grad_dev).
//
// dispatch: a stable counting sort of the live selections s = t K + k by expert,
// then xs[r] = x[src[r] / K]. combine: out[t] = sum_k w[t, k] ys[pos[t, k]] in f32,
// k ascending. Its gradient: dys[pos[t, k]] = w[t, k] dout[t], dw[t, k] = <dout[t],
// ys[pos[t, k]]>. All are bound by the rows' bytes, the small ones by their launches:
// 8192 bf16 rows of 7168 to 35000 places 134 us (4.6 TB/s, nearly the rate of a copy; counts
// and places 11 of them); combine of 32768 such rows 94 us (5.6 TB/s, mostly reads), its
// gradient 210 (5.0 TB/s); one token's rows 4.7, combine of 16 tokens 5.0, each in one launch.
#include "coli_hip_host.h"
#include "coli_rows.h"

#include "coli_backend_abi.h"
#include "coli_hip_ext.h"

#include <algorithm>

#define COLI_SORT_MAX_E 1024
#define COLI_SORT_MAX_T (1 << 23)   // a grid of 256-thread workgroups by row
#define COLI_SORT_MAX_K 64
#define COLI_SORT_FEW 4096      // selections that every workgroup places by itself
#define COLI_SORT_BLOCKS 256    // counts of at most so many workgroups are added up
#define COLI_ROW_PIECE 4096     // bytes of a row that a workgroup moves

struct SortArgs {
    const int *idx, *keff;
    const uint8_t *mask;
    int T, E, K, N;
    const uint8_t *x;
    uint8_t *xs;
    size_t rb;
    int *offsets, *src, *pos, *hist;
    int per, nblk;
    uint32_t magic;   // ceil(2^32 / K), where selections below 2^26 are divided by it; 0: divide
};

// Expert of selection s, E where it is not live.
__device__ __forceinline__ int sort_key(const SortArgs &a, int s) {
    const int t = a.magic ? (int)__umulhi((uint32_t)s, a.magic) : s / a.K, k = s - t * a.K, e = a.idx[s];
    // (every load asked for: short-circuited they would wait for one another)
    const int most = a.keff ? a.keff[t] : a.K, on = a.mask ? a.mask[t] : 1;
    const bool live = ((unsigned)e < (unsigned)a.E) & (k < most) & (on != 0);
    return live ? e : a.E;
}

// Exclusive sum over the workgroup's threads (NT of them), and the total.
template <int NT> __device__ __forceinline__ int block_scan(int v, int *tmp, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(s, o);
        if (lane >= o) s += u;
    }
    if (lane == 63) tmp[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        if (w < wave) before += tmp[w];
        total += tmp[w];
    }
    return before + s - v;
}

// One piece of row t to its places: the row is read once. A piece that would pass
// the row's end is moved back (the same bytes twice); rows below 16 bytes go by bytes.
// NT: past the caches (a template's: of two stores under a branch the compiler makes one
// and drops the hint).
template <bool NT> __device__ __forceinline__ void copy_piece(const SortArgs &a, int t, const int *place) {
    const size_t c = (size_t)blockIdx.y * COLI_ROW_PIECE + threadIdx.x * 16;
    if (c >= a.rb) return;
    const uint8_t *xr = a.x + (size_t)t * a.rb;
    if (a.rb < 16) {
        for (int k = 0; k < a.K; k++)
            if (place[k] >= 0)
                for (size_t i = 0; i < a.rb; i++) a.xs[(size_t)place[k] * a.rb + i] = xr[i];
        return;
    }
    const size_t p = min(c, a.rb - 16);
    const u32x4 v = *GPTR(u32x4a1, xr + p);
    for (int k = 0; k < a.K; k++) {
        if (place[k] < 0) continue;
        u32x4a1 *to = (u32x4a1 *)(a.xs + (size_t)place[k] * a.rb + p);
        if constexpr (NT) __builtin_nontemporal_store((u32x4a1)v, to);
        else *to = v;
    }
}

// Few selections: one launch. A workgroup (row, piece) counts, for each of its
// row's selections, those that come before it; the row behind the last one is the
// offsets'.
__global__ __launch_bounds__(256) void coli_dispatch_few(SortArgs a) {
    __shared__ int key[COLI_SORT_FEW], place[COLI_SORT_MAX_K], cnt[COLI_SORT_MAX_K], tmp[4];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (t == a.T) {
        if (blockIdx.y) return;
        int *hist = key;   // [E]
        for (int e = tid; e < COLI_SORT_MAX_E; e += 256) hist[e] = 0;
        __syncthreads();
#pragma unroll 4
        for (int s = tid; s < a.N; s += 256) {
            const int e = sort_key(a, s);
            if (e < a.E) atomicAdd(hist + e, 1);
        }
        __syncthreads();
        int v[4], sum = 0, total;
#pragma unroll
        for (int i = 0; i < 4; i++) sum += v[i] = hist[4 * tid + i];
        int at = block_scan<256>(sum, tmp, total);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (4 * tid + i < a.E) a.offsets[4 * tid + i] = at;
            at += v[i];
        }
        if (tid == 0) a.offsets[a.E] = total;
        return;
    }
    // keys by expert, then selection: one number, so a place is a count of smaller ones
#pragma unroll 4
    for (int s = tid; s < a.N; s += 256) key[s] = sort_key(a, s) * COLI_SORT_FEW + s;
    if (tid < a.K) cnt[tid] = 0;
    __syncthreads();
    for (int k0 = 0; k0 < a.K; k0 += 8) {
        int mine[8], n[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            mine[i] = __builtin_amdgcn_readfirstlane(key[t * a.K + min(k0 + i, a.K - 1)]);
            n[i] = 0;
        }
        for (int s0 = 64 * wave; s0 < a.N; s0 += 256) {
            const int o = s0 + lane < a.N ? key[s0 + lane] : 0x7fffffff;
#pragma unroll
            for (int i = 0; i < 8; i++) n[i] += __popcll(__ballot(o < mine[i]));
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (lane == 0 && k0 + i < a.K) atomicAdd(cnt + k0 + i, n[i]);
    }
    __syncthreads();
    if (tid < a.K) place[tid] = key[t * a.K + tid] < a.E * COLI_SORT_FEW ? cnt[tid] : -1;
    __syncthreads();
    if (blockIdx.y == 0 && tid < a.K) {
        const int p = place[tid];
        a.pos[t * a.K + tid] = p;
        if (p >= 0) a.src[p] = t * a.K + tid;
    }
    if (a.x) copy_piece<false>(a, t, place);
}

// Many selections: counts by workgroup and expert ...
__global__ __launch_bounds__(1024) void coli_dispatch_count(SortArgs a) {
    __shared__ int cnt[COLI_SORT_MAX_E];
    const int b = blockIdx.x, s0 = b * a.per, s1 = min(a.N, s0 + a.per);
    cnt[threadIdx.x] = 0;
    __syncthreads();
    for (int s = s0 + threadIdx.x; s < s1; s += 1024) {
        const int e = sort_key(a, s);
        if (e < a.E) atomicAdd(cnt + e, 1);
    }
    __syncthreads();
    if (threadIdx.x < a.E) a.hist[b * a.E + threadIdx.x] = cnt[threadIdx.x];
}

// ... then places. Each wave has a run of the workgroup's selections: it counts the
// run by expert, finds where its rows of each expert begin, and goes through the run
// again 64 selections at a time, a lane's rank among the equal ones by ballots.
__global__ __launch_bounds__(1024) void coli_dispatch_place(SortArgs a) {
    extern __shared__ int at[];   // [16][E]
    __shared__ int tmp[16];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int s0 = b * a.per + wave * (a.per / 16), s1 = min(min(a.N, s0 + a.per / 16), (b + 1) * a.per);
    int *mine = at + wave * a.E;
    for (int e = tid; e < 16 * a.E; e += 1024) at[e] = 0;
    // counts of the workgroups before this one and of all, 1024 / 2^lg threads an expert
    __shared__ int part[2][1024];
    int before = 0, sum = 0, total;
    const int lg = 32 - __clz(a.E - 1 | 1), e0 = tid & ((1 << lg) - 1);
    if (e0 < a.E)
#pragma unroll 8
        for (int q = tid >> lg; q < a.nblk; q += 1024 >> lg) {
            const int v = a.hist[q * a.E + e0];
            sum += v;
            before += q < b ? v : 0;
        }
    part[0][tid] = before;
    part[1][tid] = sum;
    __syncthreads();
    before = sum = 0;
    if (tid < a.E)
        for (int q = tid; q < 1024; q += 1 << lg) {
            before += part[0][q];
            sum += part[1][q];
        }
    const int first = block_scan<1024>(sum, tmp, total);
    for (int s = s0 + lane; s < s1; s += 64) {
        const int e = sort_key(a, s);
        if (e < a.E) atomicAdd(mine + e, 1);
    }
    __syncthreads();
    if (tid < a.E) {
        if (b == 0) a.offsets[tid] = first;
        int p = first + before;
#pragma unroll
        for (int w = 0; w < 16; w++) {
            const int v = at[w * a.E + tid];
            at[w * a.E + tid] = p;
            p += v;
        }
    }
    if (b == 0 && tid == 0) a.offsets[a.E] = total;
    __syncthreads();
    const int nbits = 32 - __clz(a.E);
    for (int c = s0; c < s1; c += 64) {
        const int s = c + lane;
        const int e = s < s1 ? sort_key(a, s) : a.E;
        unsigned long long same = ~0ull;
        for (int i = 0; i < nbits; i++) {
            const unsigned long long m = __ballot((e >> i) & 1);
            same &= (e >> i) & 1 ? m : ~m;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const bool live = e < a.E;
        const int p = live ? mine[e] + rank : -1;
        __builtin_amdgcn_wave_barrier();
        if (live && rank == 0) mine[e] = p + __popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (s < s1) {
            a.pos[s] = p;
            if (live) a.src[p] = s;
        }
    }
}

template <bool NT> __global__ __launch_bounds__(256) void coli_dispatch_rows(SortArgs a) {
    copy_piece<NT>(a, blockIdx.x, a.pos + (size_t)blockIdx.x * a.K);
}

// No rows: offsets of zeros.
__global__ void coli_dispatch_none(SortArgs a) {
    for (int e = threadIdx.x; e <= a.E; e += 256) a.offsets[e] = 0;
}

extern "C" int coli_hip_dispatch_dev(int device, const int *idx, const int *keff, const unsigned char *mask, int T, int E,
                                     int K, const void *x, size_t row_bytes, int *offsets, int *src, int *pos, void *xs) {
    if (fault_injected()) return 0;
    if (T < 0 || T > COLI_SORT_MAX_T || E < 1 || E > COLI_SORT_MAX_E || K < 1 || K > COLI_SORT_MAX_K ||
        (int64_t)T * K > (1 << 30) || !offsets || !x != !xs || (x && (row_bytes < 1 || row_bytes > ((size_t)64 << 20))))
        return 0;
    const size_t n4 = (size_t)T * K * 4, xb = x ? (size_t)T * row_bytes : 0;
    if (T && (!idx || !src || !pos)) return 0;
    if (!outputs_apart({{offsets, (size_t)(E + 1) * 4}, {src, n4}, {pos, n4}, {xs, xb * K}, {x, xb}, {idx, n4},
                        {keff, (size_t)T * 4}, {mask, (size_t)T}}, 4))
        return 0;
    DevCtx *ctx = ctx_of(device);
    if (!bind_ctx(ctx)) return 0;
    SortArgs a = {};
    a.idx = idx;
    a.keff = keff;
    a.mask = mask;
    a.T = T;
    a.E = E;
    a.K = K;
    a.N = T * K;
    a.x = (const uint8_t *)x;
    a.xs = (uint8_t *)xs;
    a.rb = x ? row_bytes : 0;
    a.offsets = offsets;
    a.src = src;
    a.pos = pos;
    a.magic = K > 1 && a.N < (1 << 26) ? (uint32_t)(((1ull << 32) + K - 1) / K) : 0;
    forget_emitted(ctx, offsets, (size_t)(E + 1) * 4);
    hipStream_t st = ctx->stream;
    if (!T) {
        hipLaunchKernelGGL(coli_dispatch_none, dim3(1), dim3(256), 0, st, a);
        return hip_check(hipGetLastError(), "dispatch");
    }
    forget_emitted(ctx, src, n4);
    forget_emitted(ctx, pos, n4);
    if (xs) forget_emitted(ctx, xs, xb * K);
    const unsigned pieces = x ? (unsigned)((a.rb + COLI_ROW_PIECE - 1) / COLI_ROW_PIECE) : 1;
    // (each workgroup goes through all selections: 2000 of 250 rows 7.0 us, in three launches
    // 10.6; 4000 of 500 rows 10.6 and 10.7; 2000 of 2000 rows 11.6 and 9.7)
    if (a.N <= COLI_SORT_FEW && (int64_t)a.N * T * pieces <= 1500000) {
        hipLaunchKernelGGL(coli_dispatch_few, dim3(T + 1, pieces), dim3(256), 0, st, a);
        return hip_check(hipGetLastError(), "dispatch");
    }
    a.per = std::max(1024, (a.N + COLI_SORT_BLOCKS - 1) / COLI_SORT_BLOCKS + 1023 & ~1023);
    a.nblk = (a.N + a.per - 1) / a.per;
    if (!reserve_kept(ctx, &ctx->sort_hist, (size_t)COLI_SORT_BLOCKS * COLI_SORT_MAX_E * 4, 0)) return 0;
    a.hist = (int *)ctx->sort_hist.p;
    hipLaunchKernelGGL(coli_dispatch_count, dim3(a.nblk), dim3(1024), 0, st, a);
    if (!hip_check(hipGetLastError(), "dispatch counts")) return 0;
    hipLaunchKernelGGL(coli_dispatch_place, dim3(a.nblk), dim3(1024), (size_t)16 * E * 4, st, a);
    if (!hip_check(hipGetLastError(), "dispatch places")) return 0;
    // (sorted rows beyond half of the 256 MB cache go past it)
    if (x && xb * K > ((size_t)128 << 20)) hipLaunchKernelGGL(coli_dispatch_rows<true>, dim3(T, pieces), dim3(256), 0, st, a);
    else if (x) hipLaunchKernelGGL(coli_dispatch_rows<false>, dim3(T, pieces), dim3(256), 0, st, a);
    return hip_check(hipGetLastError(), "dispatch rows");
}

// ---------------------------------------------------------------------------
// combine
// ---------------------------------------------------------------------------
struct CombineArgs {
    const void *ys, *dout;
    const int *pos;
    const float *w;
    int T, K, N, D;
    void *out, *dys;
    float *dw;
};

// One row t a workgroup and 256 x VE columns. The loads of up to KB selections are
// requested together: a place that is not live reads row 0 (one past K the last place's
// row) and counts for nothing, so no load waits behind a branch.
template <typename T, int VE, int KB, bool NT> __global__ __launch_bounds__(256) void coli_combine(CombineArgs a) {
    const int t = blockIdx.x, c0 = (blockIdx.y * 256 + threadIdx.x) * VE;
    if (c0 >= a.D) return;
    const int c = min(c0, a.D - VE);
    const int *pos = a.pos + (size_t)t * a.K;
    const float *w = a.w ? a.w + (size_t)t * a.K : nullptr;
    float acc[VE] = {};
    for (int k0 = 0; k0 < a.K; k0 += KB) {
        float v[KB][VE];
        bool live[KB];
#pragma unroll
        for (int i = 0; i < KB; i++) {
            const int p = pos[min(k0 + i, a.K - 1)];
            const bool in = (unsigned)p < (unsigned)a.N;
            live[i] = in && k0 + i < a.K;
            el_load<T, VE, NT>((const T *)a.ys + (size_t)(in ? p : 0) * a.D + c, v[i]);
        }
#pragma unroll
        for (int i = 0; i < KB; i++) {
            const float f = w ? w[min(k0 + i, a.K - 1)] : 1.0f;
#pragma unroll
            for (int j = 0; j < VE; j++) acc[j] = live[i] ? fmaf(f, v[i][j], acc[j]) : acc[j];
        }
    }
    el_store<T, VE>((T *)a.out + (size_t)t * a.D + c, acc);
}

// Gradients: a wave for each selection. Neighbours share the row of dout, which
// stays cached.
template <typename T, int VE, bool NT> __global__ __launch_bounds__(256) void coli_combine_grad(CombineArgs a) {
    const int64_t s = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (s >= (int64_t)a.T * a.K) return;
    const int lane = threadIdx.x & 63, t = (int)(s / a.K), p = a.pos[s];
    const bool live = (unsigned)p < (unsigned)a.N;
    if (!live) {
        if (a.dw && lane == 0) a.dw[s] = 0.0f;
        return;
    }
    const float f = a.w ? a.w[s] : 1.0f;
    const T *dout = (const T *)a.dout + (size_t)t * a.D, *y = (const T *)a.ys + (size_t)p * a.D;
    T *dy = (T *)a.dys + (size_t)p * a.D;
    float sum = 0.0f;
    for (int c0 = lane * VE; c0 < a.D; c0 += 64 * VE) {
        const int c = min(c0, a.D - VE);
        float g[VE], v[VE];
        el_load<T, VE>(dout + c, g);
        if (a.dw) {
            el_load<T, VE>(y + c, v);
#pragma unroll
            for (int i = 0; i < VE; i++)   // (elements that the moved-back piece has twice count once)
                sum = c + i >= c0 ? fmaf(g[i], v[i], sum) : sum;
        }
        if (a.dys) {
#pragma unroll
            for (int i = 0; i < VE; i++) g[i] *= f;
            el_store<T, VE, NT>(dy + c, g);
        }
    }
    if (!a.dw) return;
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) a.dw[s] = sum;
}

static bool combine_shape_ok(int dtype, int T, int K, int N, int D) {
    return dtype >= 0 && dtype <= 2 && T >= 0 && T <= COLI_SORT_MAX_T && K >= 1 && K <= COLI_SORT_MAX_K &&
           (int64_t)T * K <= (1 << 30) && N >= 0 && D >= 1 && D <= (1 << 24);
}

// ys (and dys) beyond half of the 256 MB cache go past it: combine of 32768 bf16 rows of 7168
// 107 -> 94 us. Before and behind its gradient, as a training step has it, 122 -> 94, the
// gradient itself 185 -> 210 (it no longer finds rows of ys in the cache), the step 418 ->
// 398. Where half of the rows are live, and so half of N's bytes, the step is 256 -> 259.
// Smaller ones may be there still for whoever reads them next.
template <typename T, int VE> static void combine_launch(const CombineArgs &a, bool grad, hipStream_t st) {
    const bool nt = VE > 1 && (size_t)a.N * a.D * sizeof(T) > ((size_t)128 << 20);
    if (grad) {
        const unsigned nw = (unsigned)(((int64_t)a.T * a.K + 3) / 4), gx = std::min(nw, 1u << 16);
        const dim3 g(gx, (nw + gx - 1) / gx);
        if (nt) hipLaunchKernelGGL((coli_combine_grad<T, VE, VE != 1>), g, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((coli_combine_grad<T, VE, false>), g, dim3(256), 0, st, a);
        return;
    }
    const dim3 g(a.T, (a.D + 256 * VE - 1) / (256 * VE));
    if (nt && a.K > 4) hipLaunchKernelGGL((coli_combine<T, VE, 8, VE != 1>), g, dim3(256), 0, st, a);
    else if (nt && a.K > 1) hipLaunchKernelGGL((coli_combine<T, VE, 4, VE != 1>), g, dim3(256), 0, st, a);
    else if (nt) hipLaunchKernelGGL((coli_combine<T, VE, 1, VE != 1>), g, dim3(256), 0, st, a);
    else if (a.K == 1) hipLaunchKernelGGL((coli_combine<T, VE, 1, false>), g, dim3(256), 0, st, a);
    else if (a.K == 2) hipLaunchKernelGGL((coli_combine<T, VE, 2, false>), g, dim3(256), 0, st, a);
    else if (a.K <= 4) hipLaunchKernelGGL((coli_combine<T, VE, 4, false>), g, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((coli_combine<T, VE, 8, false>), g, dim3(256), 0, st, a);
}
template <typename T> static void combine_run(const CombineArgs &a, bool grad, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (a.D >= V) combine_launch<T, V>(a, grad, st);
    else combine_launch<T, 1>(a, grad, st);
}
static int combine_call(DevCtx *ctx, const CombineArgs &a, int dtype, bool grad) {
    if (dtype == 0) combine_run<float>(a, grad, ctx->stream);
    else if (dtype == 1) combine_run<_Float16>(a, grad, ctx->stream);
    else combine_run<__bf16>(a, grad, ctx->stream);
    return hip_check(hipGetLastError(), grad ? "combine gradient" : "combine");
}

// No place is inside: zeros.
__global__ void coli_combine_none(uint8_t *out, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) out[i] = 0;
}

extern "C" int coli_hip_combine_dev(int device, const void *ys, int dtype, const int *pos, const float *w, int T, int K,
                                    int N, int D, void *out) {
    if (fault_injected()) return 0;
    if (!combine_shape_ok(dtype, T, K, N, D)) return 0;
    const size_t es = dtype ? 2 : 4, n4 = (size_t)T * K * 4, ob = (size_t)T * D * es;
    if ((T && (!pos || !out || (N && !ys))) ||
        !outputs_apart({{out, ob}, {ys, (size_t)N * D * es}, {pos, n4}, {w, n4}}, 1))
        return 0;
    DevCtx *ctx = ctx_of(device);
    if (!bind_ctx(ctx)) return 0;
    if (!T) return 1;
    forget_emitted(ctx, out, ob);
    CombineArgs a = {};
    a.ys = ys;
    a.pos = pos;
    a.w = w;
    a.T = T;
    a.K = K;
    a.N = N;
    a.D = D;
    a.out = out;
    if (!N) {
        hipLaunchKernelGGL(coli_combine_none, dim3((unsigned)std::min((ob + 255) / 256, (size_t)4096)), dim3(256), 0,
                           ctx->stream, (uint8_t *)out, ob);
        return hip_check(hipGetLastError(), "combine");
    }
    return combine_call(ctx, a, dtype, false);
}

extern "C" int coli_hip_combine_grad_dev(int device, const void *ys, int dtype, const int *pos, const float *w,
                                         const void *dout, int T, int K, int N, int D, void *dys, float *dw) {
    if (fault_injected()) return 0;
    if (!combine_shape_ok(dtype, T, K, N, D) || (!dys && !dw)) return 0;
    const size_t es = dtype ? 2 : 4, n4 = (size_t)T * K * 4, yb = (size_t)N * D * es;
    if ((T && (!pos || !dout || (N && dw && !ys))) ||
        !outputs_apart({{dys, yb}, {dw, n4}, {ys, yb}, {dout, (size_t)T * D * es}, {pos, n4}, {w, n4}}, 2))
        return 0;
    DevCtx *ctx = ctx_of(device);
    if (!bind_ctx(ctx)) return 0;
    if (!T) return 1;
    if (dys) forget_emitted(ctx, dys, yb);
    if (dw) forget_emitted(ctx, dw, n4);
    CombineArgs a = {};
    a.ys = ys;
    a.dout = dout;
    a.pos = pos;
    a.w = w;
    a.T = T;
    a.K = K;
    a.N = N;
    a.D = D;
    a.dys = dys;
    a.dw = dw;
    return combine_call(ctx, a, dtype, true);
}
