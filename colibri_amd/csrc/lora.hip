// lora.hip -- low-rank adapters of many requests beside a resident projection.
//
// Row s of a call carries an adapter slot a (or none):
//   forward   y[s] = W x[s] + scale_a B_a (A_a x[s])
//   backward  h = A_a x, dh = scale_a B_a^T dy;  dA_a = sum_s dh[s] x[s]^T,
//             dB_a = scale_a sum_s dy[s] h[s]^T,  dx[s] = W^T dy[s] + A_a^T dh[s]
//
// The bank keeps both factors with the long dimension contiguous, V = A
// [rank][I] and V = B^T [rank][O], so three kernels do all of it:
//   shrink  h[s][r]   = sum_n X[s][n] V[r][n]        (A x, B^T dy)
//   expand  Y[s][n]  += scale sum_r h[s][r] V[r][n]  (B h, A^T dh)
//   outer   G[r][n]   = scale sum_s h[s][r] X[s][n]  (dA, dB)
// on v_mfma_f32_16x16x4_f32: the adapters' products are a few hundredths of
// the projection's, so f32 operands cost nothing that the rows' bytes do not
// hide, and need neither splitting nor exponents. Rows of one slot are
// gathered 16 at a time into an MFMA tile: up to 64 rows each workgroup finds
// its tile with one ballot over the rows' slots, beyond it a one-workgroup
// stable counting sort lists them. Sums run in a fixed order.
#include "coli_hip_host.h"
#include "coli_device.h"

#include "coli_backend_abi.h"
#include "coli_hip_ext.h"

#include <algorithm>
#include <cmath>
#include <cstdlib>

#define COLI_LORA_MAX_SLOTS 1024
#define COLI_LORA_MAX_RANK 256
#define COLI_LORA_BALLOT 64      // rows a workgroup groups by itself
#define COLI_LORA_TILE 16        // rows of a tile

struct LoraMeta {
    int rank;
    float scale;
};

struct ColiHipLora {
    int device, I, O, slots, max_rank, dtype;
    int Rp, Ip, Op;              // rank rounded up to 16, 32 or a multiple of 64, I and O to 64: padding is zero
    void *a, *bt;                // [slots][Rp][Ip], [slots][Rp][Op]
    LoraMeta *meta;              // [slots]; rank 0: nothing set
};

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// Eight consecutive factors as f32 (16-byte aligned).
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const floatx4 a = *GPTR(floatx4, p), b = *GPTR(floatx4, p + 4);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[i] = a[i];
        v[4 + i] = b[i];
    }
}
__device__ __forceinline__ void load8(const _Float16 *p, float (&v)[8]) {
    const half8v a = *GPTR(half8v, p);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (float)a[i];
}
struct bf16_t {
    uint16_t bits;
};
__device__ __forceinline__ void load8(const bf16_t *p, float (&v)[8]) {
    const u16x8 a = *GPTR(u16x8, p);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __uint_as_float((uint32_t)a[i] << 16);
}

// ---------------------------------------------------------------------------
// the bank
// ---------------------------------------------------------------------------
// Copies an adapter into its slot: workgroups [0, na) write the rows of A,
// 2048 columns each, the others 64 x 64 blocks of B transposed through LDS.
template <typename T>
__global__ __launch_bounds__(256) void coli_lora_set(const T *__restrict__ a, const T *__restrict__ b, T *__restrict__ va,
                                                     T *__restrict__ vb, LoraMeta *meta, int rank, float scale, int I,
                                                     int O, int Ip, int Op, int Rp, int na, int ca) {
    const int tid = threadIdx.x;
    if (blockIdx.x == 0 && tid == 0) *meta = {rank, scale};
    if ((int)blockIdx.x < na) {
        const int r = blockIdx.x / ca, c0 = (blockIdx.x - r * ca) * 2048;
        for (int c = c0 + tid; c < min(Ip, c0 + 2048); c += 256)
            va[(size_t)r * Ip + c] = r < rank && c < I ? a[(size_t)r * I + c] : T{};
        return;
    }
    __shared__ T tile[64][66];
    const int nb = blockIdx.x - na, no = Op / 64, o0 = (nb % no) * 64, r0 = (nb / no) * 64;
    for (int k = tid; k < 4096; k += 256) {
        const int o = o0 + (k >> 6), r = r0 + (k & 63);
        tile[k >> 6][k & 63] = o < O && r < rank ? b[(size_t)o * rank + r] : T{};
    }
    __syncthreads();
    for (int k = tid; k < 4096; k += 256) {
        const int r = r0 + (k >> 6);
        if (r < Rp) vb[(size_t)r * Op + o0 + (k & 63)] = tile[k & 63][k >> 6];
    }
}

// ---------------------------------------------------------------------------
// rows by slot
// ---------------------------------------------------------------------------
struct LoraRows {
    const int *slot;             // [S]
    const LoraMeta *meta;
    int S, slots;
    // beyond COLI_LORA_BALLOT rows (coli_lora_sort): rows in slot order, each
    // slot's run in it, and the tiles (slot, first, rows)
    int *perm;                   // [S]
    int2 *run;                   // [slots]: first, rows
    int4 *tile;                  // [ntile]
    int *ntile;
};

__device__ __forceinline__ bool lora_live(const LoraRows &w, int s) {
    return s >= 0 && s < w.slots && w.meta[s].rank > 0;
}

// Tile t of the call into LDS rows[]: the slot, and its rows' number (0: no
// such tile). Every wave calls it; the caller synchronizes.
__device__ __forceinline__ int lora_tile(const LoraRows &w, int t, int *rows, int &slot) {
    const int lane = threadIdx.x & 63;
    if (w.S <= COLI_LORA_BALLOT) {
        // tile t starts at row t: the row must be its slot's 1st, 17th, ... one
        const int s = lane < w.S ? w.slot[lane] : -1;
        const bool live = lora_live(w, s);
        slot = __builtin_amdgcn_readlane(live ? s : -1, t);
        if (slot < 0) return 0;
        const unsigned long long m = __builtin_amdgcn_ballot_w64(live && s == slot);
        const int first = __popcll(m & ((1ull << t) - 1ull));
        if (first % COLI_LORA_TILE) return 0;
        const int at = __popcll(m & ((1ull << lane) - 1ull)) - first;
        if ((m >> lane & 1) && at >= 0 && at < COLI_LORA_TILE) rows[at] = lane;
        return min(COLI_LORA_TILE, __popcll(m) - first);
    }
    if (t >= *w.ntile) return 0;
    const int4 e = w.tile[t];
    slot = e.x;
    if (lane < e.z) rows[lane] = w.perm[e.y + lane];
    return e.z;
}

// Stable counting sort of the rows by slot: eight waves count and then place a
// run of rows each, 64 at a time, so a slot's rows keep their order (the sums
// over them do not depend on timing).
__global__ __launch_bounds__(512) void coli_lora_sort(LoraRows w) {
    extern __shared__ int cnt[];   // [8][slots]
    __shared__ int wsum[8][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nsl = w.slots;
    const int per = ((w.S + 7) / 8 + 63) & ~63, r0 = wave * per, r1 = min(w.S, r0 + per);
    for (int k = tid; k < 8 * nsl; k += 512) cnt[k] = 0;
    __syncthreads();
    int *mine = cnt + wave * nsl;
    auto slot_of = [&](int r) {
        const int s = r < r1 ? w.slot[r] : -1;
        return lora_live(w, s) ? s : -1;
    };
    for (int r = r0; r < r1; r += 64) {
        const int s = slot_of(r + lane);
        unsigned long long todo = __builtin_amdgcn_ballot_w64(s >= 0);
        while (todo) {
            const int sl = __builtin_amdgcn_readlane(s, __builtin_ctzll(todo));
            const unsigned long long m = __builtin_amdgcn_ballot_w64(s == sl);
            if (lane == 0) mine[sl] += __popcll(m);
            todo &= ~m;
        }
    }
    __syncthreads();
    // exclusive sums over (slot, wave), of the rows and of the tiles
    int base = 0, tbase = 0;
    for (int c0 = 0; c0 < nsl; c0 += 512) {
        const int s = c0 + tid;
        int n = 0;
        if (s < nsl)
            for (int v = 0; v < 8; v++) n += cnt[v * nsl + s];
        const int nt = (n + COLI_LORA_TILE - 1) / COLI_LORA_TILE;
        int x = n, y = nt;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int px = __shfl_up(x, o), py = __shfl_up(y, o);
            if (lane >= o) {
                x += px;
                y += py;
            }
        }
        if (lane == 63) {
            wsum[wave][0] = x;
            wsum[wave][1] = y;
        }
        __syncthreads();
        int bx = base, by = tbase;
        for (int v = 0; v < 8; v++) {
            if (v < wave) {
                bx += wsum[v][0];
                by += wsum[v][1];
            }
            base += wsum[v][0];
            tbase += wsum[v][1];
        }
        if (s < nsl) {
            const int first = bx + x - n, t0 = by + y - nt;
            w.run[s] = make_int2(first, n);
            for (int k = 0; k < nt; k++)
                w.tile[t0 + k] = make_int4(s, first + k * COLI_LORA_TILE, min(COLI_LORA_TILE, n - k * COLI_LORA_TILE), 0);
            int at = first;
            for (int v = 0; v < 8; v++) {
                const int c = cnt[v * nsl + s];
                cnt[v * nsl + s] = at;
                at += c;
            }
        }
        __syncthreads();
    }
    if (tid == 0) *w.ntile = tbase;
    for (int r = r0; r < r1; r += 64) {
        const int s = slot_of(r + lane);
        unsigned long long todo = __builtin_amdgcn_ballot_w64(s >= 0);
        while (todo) {
            const int sl = __builtin_amdgcn_readlane(s, __builtin_ctzll(todo));
            const unsigned long long m = __builtin_amdgcn_ballot_w64(s == sl);
            const int at = mine[sl];
            if (s == sl) w.perm[at + __popcll(m & ((1ull << lane) - 1ull))] = r + lane;
            if (lane == 0) mine[sl] = at + __popcll(m);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the other lanes read it next
            todo &= ~m;
        }
    }
}

// ---------------------------------------------------------------------------
// the three products
// ---------------------------------------------------------------------------
template <typename T> struct LoraSide {
    const float *x;              // [S][N] rows (shrink and outer: read; expand: y)
    const T *v;                  // [slots][Rp][Np]
    float *h;                    // [splits][S][Rp] shrunk rows
    float *out;                  // expand: y [S][N]; outer: the gradient
    int N, Np, splits;
    int vec;                     // N % 4 == 0 and rows 16-byte aligned
};

// Eight floats of a row from column n on, zeros past N.
__device__ __forceinline__ void row8(const float *xr, int n, int N, int vec, float (&v)[8]) {
    if (vec && n + 8 <= N) {
        load8(xr + n, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = n + i < N ? xr[n + i] : 0.0f;
    }
}

// shrink: workgroup (tile, column split, NR rank tiles of one side). The four
// waves take 32 columns in turn: lane (m, k) reads eight columns of row m and
// of factor m, which feed eight MFMAs (the order of the columns inside a sum
// is free).
template <typename T, int NR>
__global__ __launch_bounds__(256) void coli_lora_shrink(LoraRows w, LoraSide<T> s0, LoraSide<T> s1, int Rp, int nz) {
    __shared__ int rows[COLI_LORA_TILE];
    __shared__ float red[4][NR][16][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, kq = lane >> 4;
    int slot = 0;
    const int n = lora_tile(w, blockIdx.x, rows, slot);
    if (n == 0) return;   // (uniform over the workgroup)
    const LoraSide<T> s = (int)blockIdx.z < nz ? s0 : s1;
    const int rt0 = (blockIdx.z % nz) * NR, sp = blockIdx.y;
    if (sp >= s.splits || 16 * rt0 >= w.meta[slot].rank) return;
    __syncthreads();
    const int steps = (s.N + 31) / 32, per = (steps + s.splits - 1) / s.splits;
    const int k1 = min(steps, (sp + 1) * per);
    const float *xr = s.x + (size_t)rows[min(m, n - 1)] * s.N;
    const T *vr = s.v + ((size_t)slot * Rp + 16 * rt0 + m) * s.Np;
    floatx4 acc[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) acc[r] = (floatx4){0.f, 0.f, 0.f, 0.f};
    for (int k = sp * per + wave; k < k1; k += 4) {
        const int c = 32 * k + 8 * kq;
        float xv[8], vv[NR][8];
        row8(xr, c, s.N, s.vec, xv);
#pragma unroll
        for (int r = 0; r < NR; r++) load8(vr + (size_t)16 * r * s.Np + min(c, s.Np - 8), vv[r]);
#pragma unroll
        for (int r = 0; r < NR; r++)
#pragma unroll
            for (int j = 0; j < 8; j++) acc[r] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[j], vv[r][j], acc[r], 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int i = 0; i < 4; i++) red[wave][r][4 * kq + i][m] = acc[r][i];
    __syncthreads();
    for (int e = threadIdx.x; e < NR * 256; e += 256) {
        const int r = e >> 8, row = (e >> 4) & 15, c = e & 15;
        if (row < n)
            s.h[((size_t)sp * w.S + rows[row]) * Rp + 16 * (rt0 + r) + c] =
                (red[0][r][row][c] + red[1][r][row][c]) + (red[2][r][row][c] + red[3][r][row][c]);
    }
}

// scale h of one row's rank r: the column splits joined in order; zero past
// the adapter's rank.
__device__ __forceinline__ float lora_h(const float *h, int splits, size_t pitch, int r, int rank, float scale) {
    if (r >= rank) return 0.0f;
    float v = h[r];
    for (int p = 1; p < splits; p++) v += h[p * pitch + r];
    return v * scale;
}

// expand: workgroup (tile, 512 columns), a wave 128 of them: lane (m, k) holds
// row m's h of rank 4 q + k and eight columns of the factor, eight MFMAs a
// step of four ranks. The lane's results are eight consecutive columns of four
// rows, added to y.
template <typename T>
__global__ __launch_bounds__(256) void coli_lora_expand(LoraRows w, LoraSide<T> s, int Rp) {
    extern __shared__ float hs[];   // [16][Rp + 1]
    __shared__ int rows[COLI_LORA_TILE];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, kq = lane >> 4;
    int slot = 0;
    const int n = lora_tile(w, blockIdx.x, rows, slot);
    if (n == 0) return;   // (uniform over the workgroup)
    __syncthreads();
    const LoraMeta meta = w.meta[slot];
    const int rank = min(meta.rank, Rp), r4 = (rank + 3) & ~3;
    for (int e = threadIdx.x; e < 16 * r4; e += 256) {
        const int row = e / r4, r = e - row * r4;
        hs[row * (Rp + 1) + r] = row < n ? lora_h(s.h + (size_t)rows[row] * Rp, s.splits, (size_t)w.S * Rp, r, rank, meta.scale) : 0.0f;
    }
    __syncthreads();
    const int c = blockIdx.y * 512 + wave * 128 + 8 * m;
    if (blockIdx.y * 512 + wave * 128 >= s.Np) return;
    const T *vr = s.v + (size_t)slot * Rp * s.Np + min(c, s.Np - 8);
    floatx4 acc[8];
#pragma unroll
    for (int j = 0; j < 8; j++) acc[j] = (floatx4){0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < r4; r += 4) {
        float vv[8];
        load8(vr + (size_t)(r + kq) * s.Np, vv);
        const float hv = hs[m * (Rp + 1) + r + kq];
#pragma unroll
        for (int j = 0; j < 8; j++) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(hv, vv[j], acc[j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = 4 * kq + i;
        if (row >= n || c >= s.N) continue;
        float *yr = s.out + (size_t)rows[row] * s.N + c;
        if (s.vec && c + 8 <= s.N) {
            floatx4 y0 = *(const floatx4 *)yr, y1 = *(const floatx4 *)(yr + 4);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                y0[j] += acc[j][i];
                y1[j] += acc[4 + j][i];
            }
            *(floatx4 *)yr = y0;
            *(floatx4 *)(yr + 4) = y1;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (c + j < s.N) yr[j] += acc[j][i];
        }
    }
}

// outer: workgroup (64 columns, slot and NR rank tiles, side); the four waves
// take 16 rows of the slot in turn, four MFMA steps of four rows, and their
// sums are joined in LDS. Side 0: dA [slots][max_rank][N]; side 1 (dB): stored
// transposed, [slots][N][max_rank]. Every element is written, zeros where a
// slot has no rows or rank.
template <typename T, int NR>
__global__ __launch_bounds__(256) void coli_lora_outer(LoraRows w, LoraSide<T> s0, LoraSide<T> s1, int Rp, int max_rank) {
    __shared__ int rows[COLI_LORA_BALLOT];
    __shared__ float red[4][64][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, kq = lane >> 4;
    const int nrp = (Rp / 16 + NR - 1) / NR, slot = blockIdx.y / nrp, rt0 = (blockIdx.y - slot * nrp) * NR;
    const bool side1 = blockIdx.z != 0;
    // (h of one side meets the rows of the other)
    const float *x = side1 ? s1.x : s0.x;
    const int N = side1 ? s1.N : s0.N, vec = side1 ? s1.vec : s0.vec;
    const float *h = side1 ? s0.h : s1.h;
    const int splits = side1 ? s0.splits : s1.splits;
    float *out = side1 ? s1.out : s0.out;
    const int c0 = blockIdx.x * 64, c = c0 + 4 * m;
    if (c0 >= N) return;
    const LoraMeta meta = w.meta[slot];
    const int rank = min(meta.rank, Rp);
    int cnt = 0, first = 0;
    if (rank > 0) {
        if (w.S <= COLI_LORA_BALLOT) {
            const unsigned long long mk = __builtin_amdgcn_ballot_w64(lane < w.S && w.slot[min(lane, w.S - 1)] == slot);
            if (mk >> lane & 1) rows[__popcll(mk & ((1ull << lane) - 1ull))] = lane;
            cnt = __popcll(mk);
        } else {
            const int2 rn = w.run[slot];
            first = rn.x;
            cnt = rn.y;
        }
    }
    __syncthreads();
    floatx4 acc[NR][4];
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[r][j] = (floatx4){0.f, 0.f, 0.f, 0.f};
    const size_t pitch = (size_t)w.S * Rp;
    for (int p0 = 16 * wave; p0 < cnt; p0 += 64) {
        float xv[4][4], hv[4][NR];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int p = p0 + 4 * u + kq;
            const bool live = p < cnt;
            const int pc = live ? p : cnt - 1;
            const int row = w.S <= COLI_LORA_BALLOT ? rows[pc] : w.perm[first + pc];
            const float *xr = x + (size_t)row * N;
            if (vec && c + 4 <= N) {
                const floatx4 t = *GPTR(floatx4, xr + c);
#pragma unroll
                for (int j = 0; j < 4; j++) xv[u][j] = live ? t[j] : 0.0f;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) xv[u][j] = live && c + j < N ? xr[c + j] : 0.0f;
            }
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const int rk = 16 * (rt0 + r) + m;
                hv[u][r] = live ? lora_h(h + (size_t)row * Rp, splits, pitch, rk, rank, meta.scale) : 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int r = 0; r < NR; r++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    acc[r][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(hv[u][r], xv[u][j], acc[r][j], 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < NR; r++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) red[wave][lane][4 * i + j] = acc[r][j][i];
        __syncthreads();
        // wave i finishes rank 4 kq + i of the tile
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
            v[j] = (red[0][lane][4 * wave + j] + red[1][lane][4 * wave + j]) +
                   (red[2][lane][4 * wave + j] + red[3][lane][4 * wave + j]);
        const int rk = 16 * (rt0 + r) + 4 * kq + wave;
        if (rk >= max_rank) continue;
        if (side1) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (c + j < N) out[((size_t)slot * N + c + j) * max_rank + rk] = v[j];
        } else {
            float *o = out + ((size_t)slot * max_rank + rk) * N + c;
            if (vec && c + 4 <= N) {
                *(floatx4 *)o = (floatx4){v[0], v[1], v[2], v[3]};
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (c + j < N) o[j] = v[j];
            }
        }
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Column splits of the shrink: enough workgroups for two a CU, each of at
// least 256 columns (two steps of its waves).
static int shrink_splits(const DevCtx *ctx, int tiles, int N) {
    const int want = (2 * (ctx->cu_count ? ctx->cu_count : 256) + tiles - 1) / tiles;
    return std::max(1, std::min(std::min(want, 32), (N + 255) / 256));
}

static int lora_tiles(int S, int slots) {
    return S <= COLI_LORA_BALLOT ? S : S / COLI_LORA_TILE + std::min(S, slots);
}

// The rows' grouping, and (beyond COLI_LORA_BALLOT rows) the launch that makes it.
static int lora_rows(DevCtx *ctx, const ColiHipLora *l, const int *slot_dev, int S, LoraRows *w) {
    *w = LoraRows{};
    w->slot = slot_dev;
    w->meta = l->meta;
    w->S = S;
    w->slots = l->slots;
    if (S <= COLI_LORA_BALLOT) return 1;
    const size_t nt = (size_t)lora_tiles(S, l->slots);
    const size_t tb = nt * sizeof(int4), rb = (size_t)l->slots * sizeof(int2), pb = (size_t)S * sizeof(int);
    if (!reserve_kept(ctx, &ctx->lora_list, tb + rb + pb + sizeof(int), 0)) return 0;
    uint8_t *p = (uint8_t *)ctx->lora_list.p;
    w->tile = (int4 *)p;
    w->run = (int2 *)(p + tb);
    w->perm = (int *)(p + tb + rb);
    w->ntile = (int *)(p + tb + rb + pb);
    hipLaunchKernelGGL(coli_lora_sort, dim3(1), dim3(512), (size_t)8 * l->slots * sizeof(int), ctx->stream, *w);
    return hip_check(hipGetLastError(), "adapter rows");
}

template <typename T>
static LoraSide<T> lora_side(const ColiHipLora *l, bool b, const float *x, float *h, float *out, int splits) {
    LoraSide<T> s;
    s.x = x;
    s.v = (const T *)(b ? l->bt : l->a);
    s.h = h;
    s.out = out;
    s.N = b ? l->O : l->I;
    s.Np = b ? l->Op : l->Ip;
    s.splits = splits;
    s.vec = s.N % 4 == 0 && (((uintptr_t)x | (uintptr_t)out) & 15) == 0;
    return s;
}

template <typename T>
static int launch_shrink(DevCtx *ctx, const ColiHipLora *l, const LoraRows &w, const LoraSide<T> &s0,
                         const LoraSide<T> &s1, int sides) {
    const int tiles = lora_tiles(w.S, l->slots), nrt = l->Rp / 16, sp = std::max(s0.splits, sides > 1 ? s1.splits : 1);
#define COLI_SHRINK(NR)                                                                                              \
    hipLaunchKernelGGL((coli_lora_shrink<T, NR>), dim3(tiles, sp, sides *((nrt + NR - 1) / NR)), dim3(256), 0,         \
                       ctx->stream, w, s0, s1, l->Rp, (nrt + NR - 1) / NR)
    if (nrt == 1) COLI_SHRINK(1);
    else if (nrt == 2) COLI_SHRINK(2);
    else COLI_SHRINK(4);
#undef COLI_SHRINK
    return hip_check(hipGetLastError(), "adapter shrink");
}

template <typename T>
static int launch_expand(DevCtx *ctx, const ColiHipLora *l, const LoraRows &w, const LoraSide<T> &s) {
    hipLaunchKernelGGL((coli_lora_expand<T>), dim3(lora_tiles(w.S, l->slots), (s.Np + 511) / 512), dim3(256),
                       (size_t)16 * (l->Rp + 1) * sizeof(float), ctx->stream, w, s, l->Rp);
    return hip_check(hipGetLastError(), "adapter expand");
}

template <typename T>
static int launch_outer(DevCtx *ctx, const ColiHipLora *l, const LoraRows &w, const LoraSide<T> &s0, const LoraSide<T> &s1) {
    const int nrt = l->Rp / 16, cols = (std::max(l->I, l->O) + 63) / 64;
#define COLI_OUTER(NR)                                                                                             \
    hipLaunchKernelGGL((coli_lora_outer<T, NR>), dim3(cols, l->slots *((nrt + NR - 1) / NR), 2), dim3(256), 0,       \
                       ctx->stream, w, s0, s1, l->Rp, l->max_rank)
    if (nrt == 1) COLI_OUTER(1);
    else if (nrt == 2) COLI_OUTER(2);
    else COLI_OUTER(4);
#undef COLI_OUTER
    return hip_check(hipGetLastError(), "adapter gradients");
}

template <typename T>
static int lora_forward(DevCtx *ctx, ColiCudaTensor *t, const ColiHipLora *l, float *y, const float *x, int S,
                        const int *slot_dev) {
    LoraRows w;
    const int splits = shrink_splits(ctx, lora_tiles(S, l->slots), l->I);
    if (!reserve_kept(ctx, &ctx->lora_h, (size_t)splits * S * l->Rp * sizeof(float), 0) ||
        !lora_rows(ctx, l, slot_dev, S, &w))
        return 0;
    float *h = (float *)ctx->lora_h.p;
    const LoraSide<T> a = lora_side<T>(l, false, x, h, nullptr, splits);
    LoraSide<T> b = lora_side<T>(l, true, nullptr, h, y, splits);
    return launch_shrink<T>(ctx, l, w, a, a, 1) && gemm_dev(ctx, t, y, x, S) && launch_expand<T>(ctx, l, w, b);
}

template <typename T>
static int lora_backward(DevCtx *ctx, ColiCudaTensor *t, const ColiHipLora *l, const float *x, const float *dy, int S,
                         const int *slot_dev, float *dx, float *da, float *db) {
    LoraRows w;
    const int tiles = lora_tiles(S, l->slots);
    const int spa = shrink_splits(ctx, 2 * tiles, l->I), spb = shrink_splits(ctx, 2 * tiles, l->O);
    const size_t hb = (size_t)S * l->Rp * sizeof(float);
    if (!reserve_kept(ctx, &ctx->lora_h, (spa + spb) * hb, 0) || !lora_rows(ctx, l, slot_dev, S, &w)) return 0;
    float *ha = (float *)ctx->lora_h.p, *hb_ = (float *)((uint8_t *)ctx->lora_h.p + spa * hb);
    const LoraSide<T> sa = lora_side<T>(l, false, x, ha, da, spa), sb = lora_side<T>(l, true, dy, hb_, db, spb);
    if (!launch_shrink<T>(ctx, l, w, sa, sb, 2) || !launch_outer<T>(ctx, l, w, sa, sb)) return 0;
    if (!dx) return 1;
    LoraSide<T> e = lora_side<T>(l, false, nullptr, hb_, dx, spb);
    return gemm_t_dev(ctx, t, dx, dy, S) && launch_expand<T>(ctx, l, w, e);
}

// ---------------------------------------------------------------------------
// entry points
// ---------------------------------------------------------------------------
extern "C" void coli_hip_lora_free(ColiHipLora *l) {
    if (!l) return;
    DevCtx *ctx = ctx_of(l->device);
    if (ctx) {
        bind_ctx(ctx);
        (void)hipStreamSynchronize(ctx->stream);
    }
    if (l->a) (void)hipFree(l->a);
    if (l->bt) (void)hipFree(l->bt);
    if (l->meta) (void)hipFree(l->meta);
    std::free(l);
}

extern "C" int coli_hip_lora_create(ColiHipLora **out, int device, int I, int O, int slots, int max_rank, int dtype) {
    if (!out || I < 1 || O < 1 || I > (1 << 20) || O > (1 << 20) || slots < 1 || slots > COLI_LORA_MAX_SLOTS ||
        max_rank < 1 || max_rank > COLI_LORA_MAX_RANK || dtype < 0 || dtype > 2)
        return 0;
    DevCtx *ctx = ctx_of(device);
    if (!bind_ctx(ctx)) return 0;
    ColiHipLora *l = (ColiHipLora *)std::calloc(1, sizeof(ColiHipLora));
    if (!l) return 0;
    l->device = device;
    l->I = I;
    l->O = O;
    l->slots = slots;
    l->max_rank = max_rank;
    l->dtype = dtype;
    l->Rp = max_rank <= 16 ? 16 : max_rank <= 32 ? 32 : (max_rank + 63) / 64 * 64;   // whole NR passes
    l->Ip = (I + 63) / 64 * 64;
    l->Op = (O + 63) / 64 * 64;
    const size_t es = dtype ? 2 : 4, ab = (size_t)slots * l->Rp * l->Ip * es, bb = (size_t)slots * l->Rp * l->Op * es;
    // cleared: what lies past a rank is multiplied with zeros and must be finite
    if (!hip_check(hipMalloc(&l->a, ab), "adapter bank") || !hip_check(hipMalloc(&l->bt, bb), "adapter bank") ||
        !hip_check(hipMalloc((void **)&l->meta, slots * sizeof(LoraMeta)), "adapter bank") ||
        !hip_check(hipMemset(l->a, 0, ab), "adapter bank clear") ||
        !hip_check(hipMemset(l->bt, 0, bb), "adapter bank clear") ||
        !hip_check(hipMemset(l->meta, 0, slots * sizeof(LoraMeta)), "adapter bank clear") ||
        !hip_check(hipDeviceSynchronize(), "adapter bank clear")) {
        coli_hip_lora_free(l);
        return 0;
    }
    *out = l;
    return 1;
}

template <typename T>
static int lora_set(DevCtx *ctx, ColiHipLora *l, int slot, const void *a, const void *b, int rank, float scale) {
    const int ca = (l->Ip + 2047) / 2048, na = l->Rp * ca, nb = l->Op / 64 * ((l->Rp + 63) / 64);
    hipLaunchKernelGGL((coli_lora_set<T>), dim3(na + nb), dim3(256), 0, ctx->stream, (const T *)a, (const T *)b,
                       (T *)l->a + (size_t)slot * l->Rp * l->Ip, (T *)l->bt + (size_t)slot * l->Rp * l->Op, l->meta + slot,
                       rank, scale, l->I, l->O, l->Ip, l->Op, l->Rp, na, ca);
    return hip_check(hipGetLastError(), "adapter set");
}

extern "C" int coli_hip_lora_set_dev(ColiHipLora *l, int slot, const void *a_dev, const void *b_dev, int rank, float scale) {
    if (!l || slot < 0 || slot >= l->slots || rank < 0 || rank > l->max_rank || (rank && (!a_dev || !b_dev))) return 0;
    DevCtx *ctx = ctx_of(l->device);
    if (!bind_ctx(ctx)) return 0;
    if (l->dtype == 0) return lora_set<float>(ctx, l, slot, a_dev, b_dev, rank, scale);
    return lora_set<uint16_t>(ctx, l, slot, a_dev, b_dev, rank, scale);
}

static DevCtx *lora_ctx(const ColiCudaTensor *t, const ColiHipLora *l, int S) {
    if (!l || !tensor_computable(t) || S < 1 || S > COLI_GRAD_MAX_ROWS || l->device != t->device || l->I != t->I ||
        l->O != t->O)
        return nullptr;
    DevCtx *ctx = ctx_of(l->device);
    return bind_ctx(ctx) ? ctx : nullptr;
}

extern "C" int coli_hip_lora_gemm_dev(ColiCudaTensor *t, ColiHipLora *l, float *y_dev, const float *x_dev, int S,
                                      const int *slot_dev) {
    if (fault_injected()) return 0;
    if (!y_dev || !x_dev || !slot_dev) return 0;
    DevCtx *ctx = lora_ctx(t, l, S);
    if (!ctx) return 0;
    switch (l->dtype) {
    case 0: return lora_forward<float>(ctx, t, l, y_dev, x_dev, S, slot_dev);
    case 1: return lora_forward<_Float16>(ctx, t, l, y_dev, x_dev, S, slot_dev);
    default: return lora_forward<bf16_t>(ctx, t, l, y_dev, x_dev, S, slot_dev);
    }
}

extern "C" int coli_hip_lora_grad_dev(ColiCudaTensor *t, ColiHipLora *l, const float *x_dev, const float *dy_dev, int S,
                                      const int *slot_dev, float *dx_dev, float *da_dev, float *db_dev) {
    if (fault_injected()) return 0;
    if (!x_dev || !dy_dev || !slot_dev || !da_dev || !db_dev) return 0;
    DevCtx *ctx = lora_ctx(t, l, S);
    if (!ctx) return 0;
    forget_emitted(ctx, da_dev, (size_t)l->slots * l->max_rank * l->I * sizeof(float));
    forget_emitted(ctx, db_dev, (size_t)l->slots * l->max_rank * l->O * sizeof(float));
    switch (l->dtype) {
    case 0: return lora_backward<float>(ctx, t, l, x_dev, dy_dev, S, slot_dev, dx_dev, da_dev, db_dev);
    case 1: return lora_backward<_Float16>(ctx, t, l, x_dev, dy_dev, S, slot_dev, dx_dev, da_dev, db_dev);
    default: return lora_backward<bf16_t>(ctx, t, l, x_dev, dy_dev, S, slot_dev, dx_dev, da_dev, db_dev);
    }
}
