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
// the projection's, and f32 operands need neither splitting nor exponents; only
// the shrink of bf16 factors, where f32 MFMAs are most of the time at high ranks,
// splits x into three bf16 (shrink_products). Rows of one slot are
// gathered 16 at a time into an MFMA tile: up to 64 rows each workgroup finds
// its tile with one ballot over the rows' slots, beyond it a one-workgroup
// stable counting sort lists them. Sums run in a fixed order.
//
// All three are bound by the rows' bytes once there are many, by the latency of
// a launch (2 to 3 us) and of its few dependent loads up to 64. Measured (bf16
// factors; MI355X, a large copy 4.7 TB/s):
//   2048 rows, 4096 -> 14336, rank 32: both shrinks of the backward 38 us (151
//     MB, 4.0 TB/s), outer 52 us (the same rows again, 2.9 TB/s), expand 53 us
//     forward (235 MB, 4.4 TB/s) and 21 us backward (67 MB)
//   1024 rows, 14336 -> 4096, rank 64: shrink 22 us (89 MB; fp16 and f32 factors,
//     on f32 MFMAs, 40 and 41), expand 21 us
//   16 rows of 16 adapters, 7168 -> 2048, rank 32: 5.4 and 5.6 us
//   one row, 4096 -> 14336, rank 16: 4.4 and 4.2 us beside a projection of 10
// up to 64 rows the gradients' outer and the expand are one launch
// (coli_lora_finish), and the projection's row operands are built in the
// shrink's; beyond, beside the sort.
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

struct bf16_t {
    uint16_t bits;
};

// Eight consecutive factors as loaded, and as f32.
template <typename T> struct Raw8 {
    u32x4 w;
    __device__ void load(const T *p) { w = *GPTR(u32x4, p); }
    __device__ void set(const T *p) { w = *(const u32x4 *)p; }
    __device__ float get(int i) const {
        const uint32_t v = w[i >> 1];
        if constexpr (sizeof(T) == 2 && !__is_same(T, _Float16))
            return __uint_as_float(i & 1 ? v & 0xffff0000u : v << 16);
        else
            return (float)__builtin_bit_cast(half2v, v)[i & 1];
    }
};
template <> struct Raw8<float> {
    floatx4 a, b;
    __device__ void load(const float *p) {
        a = *GPTR(floatx4, p);
        b = *GPTR(floatx4, p + 4);
    }
    __device__ void set(const float *p, const float *q) {
        a = *(const floatx4 *)p;
        b = *(const floatx4 *)q;
    }
    __device__ float get(int i) const { return i < 4 ? a[i & 3] : b[i & 3]; }
};

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
        T v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int c = c0 + tid + 256 * k;
            v[k] = r < rank && c < I ? a[(size_t)r * I + c] : T{};
        }
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (c0 + tid + 256 * k < Ip) va[(size_t)r * Ip + c0 + tid + 256 * k] = v[k];
        return;
    }
    __shared__ T tile[64][66];
    const int nb = blockIdx.x - na, no = Op / 64, o0 = (nb % no) * 64, r0 = (nb / no) * 64;
    const int nr = min(64, Rp - r0);   // 16, 32 or 64: a wave's lanes cover 64 / nr rows of B
    const int sh = nr == 16 ? 4 : nr == 32 ? 5 : 6;
    T v[16];
#pragma unroll
    for (int k = 0; k < 16; k++) {
        const int e = tid + 256 * k, o = o0 + (e >> sh), r = r0 + (e & (nr - 1));
        v[k] = e < 64 * nr && o < O && r < rank ? b[(size_t)o * rank + r] : T{};
    }
#pragma unroll
    for (int k = 0; k < 16; k++)
        if (tid + 256 * k < 64 * nr) tile[(tid + 256 * k) >> sh][(tid + 256 * k) & (nr - 1)] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; k++) {
        const int e = tid + 256 * k, r = e >> 6;
        if (r < nr) vb[(size_t)(r0 + r) * Op + o0 + (e & 63)] = tile[e & 63][r];
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
    int2 *run;                   // [slots + 1]: first, rows; the last: rows without an adapter
    int4 *tile;                  // [ntile[1]], the first ntile[0] of them of slots
    int *ntile;
};

// (an empty slot counts: its rank of 0 is met where the factors are)
__device__ __forceinline__ bool lora_live(const LoraRows &w, int s) { return s >= 0 && s < w.slots; }

// Tile t of the call into LDS rows[]: the slot, and its rows' number (0: no
// such tile). Every wave calls it; the caller synchronizes. ALL: rows without
// an adapter make tiles too (up to COLI_LORA_BALLOT rows one each), of slot -1.
template <bool ALL = false>
__device__ __forceinline__ int lora_tile(const LoraRows &w, int t, int *rows, int &slot) {
    const int lane = threadIdx.x & 63;
    if (w.S <= COLI_LORA_BALLOT) {
        // tile t starts at row t: the row must be its slot's 1st, 17th, ... one
        const int s = lane < w.S ? w.slot[lane] : -1;
        const bool live = lora_live(w, s);
        slot = __builtin_amdgcn_readlane(live ? s : -1, t);
        if (slot < 0) {
            if (ALL) rows[0] = t;
            return ALL ? 1 : 0;
        }
        const unsigned long long m = __builtin_amdgcn_ballot_w64(live && s == slot);
        const int first = __popcll(m & ((1ull << t) - 1ull));
        if (first % COLI_LORA_TILE) return 0;
        const int at = __popcll(m & ((1ull << lane) - 1ull)) - first;
        if ((m >> lane & 1) && at >= 0 && at < COLI_LORA_TILE) rows[at] = lane;
        return min(COLI_LORA_TILE, __popcll(m) - first);
    }
    if (t >= w.ntile[ALL]) return 0;
    const int4 e = w.tile[t];
    slot = e.x < w.slots ? e.x : -1;
    if (lane < e.z) rows[lane] = w.perm[e.y + lane];
    return e.z;
}

// Stable counting sort of the rows by slot: NW waves count and then place a
// run of rows each, 64 at a time, so a slot's rows keep their order (the sums
// over them do not depend on timing). One workgroup (5.9 us for 841 rows, 10 us
// for 2048): the workgroups past it build the product's row operands meanwhile
// (`ride` the forward's, else `tride` the input gradient's, which takes 1024
// threads).
template <int NW>
__global__ __launch_bounds__(64 * NW) void coli_lora_sort(LoraRows w, ColiPrepArgs ride, ColiTPrepArgs tride) {
    extern __shared__ int cnt[];   // [NW][slots + 1]
    if (blockIdx.x) {
        const int b = blockIdx.x - 1;
        if (ride.nblocks) prep_frag_block<64 * NW>(ride, min(b * (NW / 4) + ((int)threadIdx.x >> 8), ride.nblocks - 1));
        else if constexpr (NW == 16) coli_t_prep_block(tride, b);
        return;
    }
    __shared__ int wsum[NW][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nsl = w.slots + 1;
    const int per = ((w.S + NW - 1) / NW + 63) & ~63, r0 = wave * per, r1 = min(w.S, r0 + per);
    for (int k = tid; k < NW * nsl; k += 64 * NW) cnt[k] = 0;
    __syncthreads();
    int *mine = cnt + wave * nsl;
    auto slot_of = [&](int r) {
        if (r >= r1) return -1;
        const int s = w.slot[r];
        return lora_live(w, s) ? s : w.slots;
    };
    int nx = slot_of(r0 + lane);
    for (int r = r0; r < r1; r += 64) {
        const int s = nx;
        nx = slot_of(r + 64 + lane);   // (-1 past the run)
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
    for (int c0 = 0; c0 < nsl; c0 += 64 * NW) {
        const int s = c0 + tid;
        int n = 0;
        if (s < nsl)
            for (int v = 0; v < NW; v++) n += cnt[v * nsl + s];
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
        for (int v = 0; v < NW; v++) {
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
            if (s == w.slots) {
                w.ntile[0] = t0;
                w.ntile[1] = t0 + nt;
            }
            for (int k = 0; k < nt; k++)
                w.tile[t0 + k] = make_int4(s, first + k * COLI_LORA_TILE, min(COLI_LORA_TILE, n - k * COLI_LORA_TILE), 0);
            int at = first;
            for (int v = 0; v < NW; v++) {
                const int c = cnt[v * nsl + s];
                cnt[v * nsl + s] = at;
                at += c;
            }
        }
        __syncthreads();
    }
    nx = slot_of(r0 + lane);
    for (int r = r0; r < r1; r += 64) {
        const int s = nx;
        nx = slot_of(r + 64 + lane);   // (-1 past the run)
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
    const float *x;              // [S][N] rows (shrink, outer)
    const T *v;                  // [slots][Rp][Np]
    float *h;                    // [splits][S][Rp] shrunk rows
    float *out;                  // expand: y [S][N]; outer: the gradient
    const float *part;           // expand: y is the sum of these [parts][S][N] instead of what it holds
    int parts;
    int N, Np, splits;
    int sorted;                  // h rows are in slot order (coli_lora_join), not the call's
};

// acc[r] += x v[r] over the lane's eight columns and its neighbours', 32 in all.
// bf16 factors: x as three bf16 (truncated, 8 bits each: exact for finite x, but
// for what lies below 2^-126; an infinity becomes NaN, as in the projection's own
// operands) on v_mfma_f32_16x16x32_bf16, three MFMAs of 16 cycles where f32 takes
// eight of 32, and the factors need no conversion (1024 x 14336, rank 64: 22 us
// against the 40 of fp16 factors; all gradients of 2048 x 4096 x 14336, rank 32:
// 90 -> 83). fp16 and f32 factors would have to be split as well: here, 32 and 44
// VALU instructions for eight of them, which takes the gain; once, when the bank
// is written, for two and three times their bytes in bf16, which is not built. f32
// sums either way.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
template <typename T, int NR>
__device__ __forceinline__ void shrink_products(const float (&x)[8], const Raw8<T> (&v)[NR], floatx4 (&acc)[NR]) {
    if constexpr (__is_same(T, bf16_t)) {
        u32x4 part[3];
        float rest[8];
#pragma unroll
        for (int j = 0; j < 8; j++) rest[j] = x[j];
#pragma unroll
        for (int p = 0; p < 3; p++)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const uint32_t a = __float_as_uint(rest[j]), b = __float_as_uint(rest[j + 1]);
                part[p][j / 2] = __builtin_amdgcn_perm(b, a, 0x07060302u);   // the upper halves
                rest[j] -= __uint_as_float(a & 0xffff0000u);
                rest[j + 1] -= __uint_as_float(b & 0xffff0000u);
            }
#pragma unroll
        for (int p = 2; p >= 0; p--)
#pragma unroll
            for (int r = 0; r < NR; r++)
                acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, part[p]),
                                                                 __builtin_bit_cast(bf16x8, v[r].w), acc[r], 0, 0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int r = 0; r < NR; r++)
                acc[r] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], v[r].get(j), acc[r], 0, 0, 0);
    }
}

// shrink: workgroup (tile, column split, NR rank tiles of one side). The W
// waves take COLS columns in turn: a lane loads 16 bytes of a row of x or of
// the factor, neighbours next to each other (lanes of one MFMA operand lie in
// sixteen rows: loaded that way every 16 bytes were a cache line of their own,
// 151 MB in 70 us), and the wave turns them round in its own LDS, 16-byte
// pieces xored with their row so that the operand reads meet no bank twice.
// Lane (m, k) then holds eight columns of row m and of factor m, which feed
// eight MFMAs (the order of the columns inside a sum is free). The next step is
// requested before this one's products. With four waves, workgroups past nown
// build the projection's activation fragments.
template <typename T, int NR> struct ShrinkGeom {
    static constexpr int COLS = NR * sizeof(T) <= 8 ? 64 : 32;
    static constexpr int XP = COLS / 4, VP = COLS * (int)sizeof(T) / 16;   // 16-byte pieces a row
    static constexpr int XI = 16 * XP / 64, VI = 16 * VP / 64;             // loads of 64 lanes: x, a rank tile
    static constexpr int BYTES = 16 * 16 * (XP + NR * VP);                 // a wave's LDS
};
template <typename T, int NR, int W>
__global__ __launch_bounds__(64 * W) void coli_lora_shrink(LoraRows w, LoraSide<T> s0, LoraSide<T> s1, int Rp, int nz,
                                                           int tiles, int splits, int nown, ColiPrepArgs ride) {
    using G = ShrinkGeom<T, NR>;
    constexpr int STEP = G::COLS;
    __shared__ int rows[COLI_LORA_TILE];
    __shared__ __attribute__((aligned(16))) uint8_t turn[W][G::BYTES];
    __shared__ float red[W][16][17];
    const int b = blockIdx.x;
    if constexpr (W == 4) {
        if (b >= nown) {
            prep_frag_block(ride, b - nown);
            return;
        }
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, kq = lane >> 4;
    const int t = b % tiles, sp = b / tiles % splits, z = b / (tiles * splits);
    int slot = 0;
    const int n = lora_tile(w, t, rows, slot);
    if (n == 0) return;   // (uniform over the workgroup)
    const LoraSide<T> s = z < nz ? s0 : s1;
    const int rt0 = (z % nz) * NR;
    if (sp >= s.splits || 16 * rt0 >= w.meta[slot].rank) return;
    __syncthreads();
    const int full = s.N / STEP, per = (full + s.splits - 1) / s.splits;
    const int k0 = sp * per, k1 = min(full, k0 + per);
    const T *vs = s.v + ((size_t)slot * Rp + 16 * rt0) * s.Np;
    floatx4 acc[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) acc[r] = (floatx4){0.f, 0.f, 0.f, 0.f};
    // the lane's places in a load: row lane / pieces of each 64 / pieces rows
    const float *xp[G::XI];
    const T *vp[G::VI];
    uint8_t *xw[G::XI], *vw[G::VI];
    uint8_t *mine = turn[wave];
#pragma unroll
    for (int i = 0; i < G::XI; i++) {
        const int r = i * (64 / G::XP) + lane / G::XP, p = lane % G::XP;
        xp[i] = s.x + (size_t)rows[min(r, n - 1)] * s.N + 4 * p;
        xw[i] = mine + (r * G::XP + (p ^ (r & (G::XP - 1)))) * 16;
    }
#pragma unroll
    for (int i = 0; i < G::VI; i++) {
        const int r = i * (64 / G::VP) + lane / G::VP, p = lane % G::VP;
        vp[i] = vs + (size_t)r * s.Np + p * (16 / (int)sizeof(T));
        vw[i] = mine + 16 * 16 * G::XP + (r * G::VP + (p ^ (r & (G::VP - 1)))) * 16;
    }
    struct Step {
        f4u x[G::XI];
        u32x4 v[NR][G::VI];
    };
    auto load = [&](int k, Step &st) {
        const size_t c = (size_t)STEP * k;
#pragma unroll
        for (int i = 0; i < G::XI; i++) st.x[i] = *GPTR(f4u, xp[i] + c);
#pragma unroll
        for (int r = 0; r < NR; r++)
#pragma unroll
            for (int i = 0; i < G::VI; i++) st.v[r][i] = *GPTR(u32x4, vp[i] + (size_t)16 * r * s.Np + c);
    };
    Step st;
    if (k0 + wave < k1) load(k0 + wave, st);
    for (int k = k0 + wave; k < k1; k += W) {
#pragma unroll
        for (int i = 0; i < G::XI; i++) *(f4u *)xw[i] = st.x[i];
#pragma unroll
        for (int r = 0; r < NR; r++)
#pragma unroll
            for (int i = 0; i < G::VI; i++) *(u32x4 *)(vw[i] + r * 16 * 16 * G::VP) = st.v[r][i];
        load(min(k + W, k1 - 1), st);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the wave's other lanes' pieces
#pragma unroll
        for (int u = 0; u < STEP / 32; u++) {
            // columns 32 u + 8 kq + 0..7
            float x[8];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const floatx4 t = *(const floatx4 *)(mine + (m * G::XP + ((8 * u + 2 * kq + e) ^ (m & (G::XP - 1)))) * 16);
#pragma unroll
                for (int j = 0; j < 4; j++) x[4 * e + j] = t[j];
            }
            Raw8<T> v[NR];
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const uint8_t *vr = mine + 16 * 16 * (G::XP + r * G::VP) + m * G::VP * 16;
                auto piece = [&](int p) { return (const T *)(vr + (p ^ (m & (G::VP - 1))) * 16); };
                if constexpr (sizeof(T) == 4) v[r].set(piece(8 * u + 2 * kq), piece(8 * u + 2 * kq + 1));
                else v[r].set(piece(4 * u + kq));
            }
            shrink_products<T, NR>(x, v, acc);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // read before the next step's writes
    }
    // columns past the last whole step: the last split, 32 a wave (the factors'
    // padding is zero, the row is read as zero past N)
    if (sp == s.splits - 1) {
        const float *xr = s.x + (size_t)rows[min(m, n - 1)] * s.N;
        const T *vr = vs + (size_t)m * s.Np + 8 * kq;
        for (int c = STEP * full + 32 * wave; c < s.N; c += 32 * W) {
            float xv[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float t = xr[min(c + 8 * kq + j, s.N - 1)];
                xv[j] = c + 8 * kq + j < s.N ? t : 0.0f;
            }
            Raw8<T> v[NR];
#pragma unroll
            for (int r = 0; r < NR; r++) v[r].load(vr + (size_t)16 * r * s.Np + c);
            shrink_products<T, NR>(xv, v, acc);
        }
    }
    for (int r = 0; r < NR; r++) {
        if (r) __syncthreads();
#pragma unroll
        for (int q = 0; q < NR; q++)
            if (q == r)
#pragma unroll
                for (int i = 0; i < 4; i++) red[wave][4 * kq + i][m] = acc[q][i];
        __syncthreads();
        if (threadIdx.x < 256) {
            const int row = threadIdx.x >> 4, c = threadIdx.x & 15;
            float v = red[0][row][c];
#pragma unroll
            for (int q = 1; q < W; q++) v += red[q][row][c];
            if (row < n) s.h[((size_t)sp * w.S + rows[row]) * Rp + 16 * (rt0 + r) + c] = v;
        }
    }
}

// The column splits of h joined, the rows in slot order: [S][Rp] a side, 4 ranks
// a thread.
struct LoraJoin {
    const float *h[2];
    float *to[2];
    int splits[2];
    const int *perm;
    int S, Rp, nblocks;          // nblocks workgroups a side
};
__global__ __launch_bounds__(256) void coli_lora_join(LoraJoin j) {
    const int b = blockIdx.x, side = b >= j.nblocks, r4 = j.Rp / 4;
    const size_t e = (size_t)(b - side * j.nblocks) * 256 + threadIdx.x, p = e / r4, n = (size_t)j.S * r4;
    if (e >= n) return;
    const floatx4 *h = (const floatx4 *)(side ? j.h[1] : j.h[0]) + (size_t)j.perm[p] * r4 + e % r4;
    const int splits = side ? j.splits[1] : j.splits[0];
    floatx4 t[4];
#pragma unroll
    for (int q = 0; q < 4; q++) t[q] = h[min(q, splits - 1) * n];   // (at most four)
    floatx4 v = t[0];
#pragma unroll
    for (int q = 1; q < 4; q++)
        if (q < splits) v += t[q];
    ((floatx4 *)(side ? j.to[1] : j.to[0]))[e] = v;
}


// An element of h: the column splits joined in order, eight requested at once.
__device__ __forceinline__ float lora_h(const float *h, int splits, size_t pitch) {
    float v = 0.0f;
    for (int p0 = 0; p0 < splits; p0 += 8) {
        float t[8];
#pragma unroll
        for (int q = 0; q < 8; q++) t[q] = h[min(p0 + q, splits - 1) * pitch];
#pragma unroll
        for (int q = 0; q < 8; q++) v += p0 + q < splits ? t[q] : 0.0f;
    }
    return v;
}

// expand: workgroup (tile, 512 columns), a wave 128 of them: lane (m, k) holds
// row m's h of rank 4 q + k and eight columns of the factor, eight MFMAs a step
// of four ranks. The lane's results are eight consecutive columns of four
// rows, added to y (JOIN: to the sum of y's partial sums, also in rows without
// an adapter). Factors and y are requested before h is joined.
template <typename T, bool JOIN>
__device__ __forceinline__ void lora_expand_block(const LoraRows &w, const LoraSide<T> &s, int Rp, int tile, int cb, float *hs) {
    // hs: [16][Rp + 1]
    __shared__ int rows[COLI_LORA_TILE];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, kq = lane >> 4;
    int slot = 0;
    const int n = lora_tile<JOIN>(w, tile, rows, slot);
    if (n == 0) return;   // (uniform over the workgroup)
    const bool none = slot < 0;
    if (none) slot = 0;
    const int c0 = cb * 512 + wave * 128, c = c0 + 8 * m;
    const T *vr = s.v + (size_t)slot * Rp * s.Np + (size_t)kq * s.Np + min(c, s.Np - 8);
    Raw8<T> v[4];
#pragma unroll
    for (int q = 0; q < 4; q++) v[q].load(vr + (size_t)4 * q * s.Np);   // (Rp >= 16)
    const LoraMeta meta = w.meta[slot];
    const int rank = none ? 0 : min(meta.rank, Rp), r16 = (rank + 15) & ~15;
    if (!JOIN && rank == 0) return;
    __syncthreads();
    const bool whole = c + 8 <= s.N;
    const float *yr[4];
#pragma unroll
    for (int i = 0; i < 4; i++) yr[i] = (JOIN ? s.part : s.out) + (size_t)rows[min(4 * kq + i, n - 1)] * s.N;
    floatx4 y[4][2];
    auto load_y = [&](int p, floatx4 (&v)[4][2]) {   // (columns past N: not kept)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) v[i][e] = row4<true>(yr[i] + (size_t)p * w.S * s.N, c + 4 * e, s.N);
    };
    load_y(0, y);
    if constexpr (JOIN) {
        for (int p = 1; p < s.parts; p++) {
            floatx4 z[4][2];
            load_y(p, z);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < 2; e++) y[i][e] += z[i][e];
        }
    }
    for (int e = threadIdx.x; e < 16 * r16; e += 256) {
        const int row = e / r16, r = e - row * r16;
        // (past the rank: zeros, also where a row of infinities shrank to NaN)
        const int hr = s.sorted ? w.tile[tile].y + min(row, n - 1) : rows[min(row, n - 1)];
        const float hv = lora_h(s.h + (size_t)hr * Rp + min(r, rank - 1), s.splits, (size_t)w.S * Rp);
        hs[row * (Rp + 1) + r] = row < n && r < rank ? meta.scale * hv : 0.0f;
    }
    __syncthreads();
    if (c0 >= s.Np) return;
    floatx4 acc[8];
#pragma unroll
    for (int j = 0; j < 8; j++) acc[j] = (floatx4){0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < r16; r += 16) {
        Raw8<T> nx[4];
        const int rn = r + 16 < r16 ? r + 16 : r;
#pragma unroll
        for (int q = 0; q < 4; q++) nx[q].load(vr + (size_t)(rn + 4 * q) * s.Np);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float hv = hs[m * (Rp + 1) + r + 4 * q + kq];
#pragma unroll
            for (int j = 0; j < 8; j++) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(hv, v[q].get(j), acc[j], 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < 4; q++) v[q] = nx[q];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = 4 * kq + i;
        if (row >= n || c >= s.N) continue;
        float *to = s.out + (size_t)rows[row] * s.N + c;
        floatx4 t[2];
#pragma unroll
        for (int j = 0; j < 8; j++) t[j >> 2][j & 3] = y[i][j >> 2][j & 3] + acc[j][i];   // (rank 0: the sums of no products, 0)
        if (whole) {
            *(f4u *)to = t[0];
            *(f4u *)(to + 4) = t[1];
        } else {
#pragma unroll
            for (int j = 0; j < 7; j++)
                if (c + j < s.N) to[j] = t[j >> 2][j & 3];
        }
    }
}

// outer: workgroup (64 columns, slot and NR rank tiles, side); its W waves
// take 16 rows of the slot in turn, four MFMA steps of four rows, the next 16
// rows requested before this step's products and their numbers a step earlier;
// the waves' sums are joined in LDS. Four waves, several workgroups a CU, so that
// one's products run beside another's first loads and its join: with 16 / 8 / 4
// waves the adapter gradients of 1024 x 14336 x 4096, rank 64, 8 slots, take 135 /
// 114 / 107 us, of 2048 x 4096 x 14336, rank 32, 4 slots, 105 / 92 / 90; sixteen
// where the workgroups leave CUs idle (512 x 7168 x 2048, one slot: this kernel
// 9.0 us against 11.0). h: up to COLI_LORA_BALLOT rows
// its column splits, joined here in LDS; beyond (LIST), joined and in slot order
// already (coli_lora_join). Side 0: dA [slots][max_rank][N]; side 1 (dB): stored
// transposed, [slots][N][max_rank]. Every element is written, zeros where a slot
// has no rows or rank.
template <typename T, int NR, int W, bool LIST>
__device__ __forceinline__ void lora_outer_block(const LoraRows &w, const LoraSide<T> &s0, const LoraSide<T> &s1, int Rp,
                                                 int max_rank, int cb, int sr, bool side1) {
    __shared__ int rows[COLI_LORA_BALLOT];
    __shared__ float hl[LIST ? 1 : COLI_LORA_BALLOT][LIST ? 1 : 16 * NR + 1];
    __shared__ float red[W][64][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, kq = lane >> 4;
    const int nrp = (Rp / 16 + NR - 1) / NR, slot = sr / nrp, rt0 = (sr - slot * nrp) * NR;
    // (h of one side meets the rows of the other)
    const float *x = side1 ? s1.x : s0.x;
    const int N = side1 ? s1.N : s0.N;
    const float *h = (side1 ? s0.h : s1.h) + 16 * rt0;
    const int splits = side1 ? s0.splits : s1.splits;
    float *out = side1 ? s1.out : s0.out;
    const int c0 = cb * 64, c = c0 + 4 * m;
    if (c0 >= N) return;
    const LoraMeta meta = w.meta[slot];
    const int rank = min(meta.rank, Rp);
    int cnt = 0, first = 0;
    const int *list = rows;
    if constexpr (!LIST) {
        const unsigned long long mk = __builtin_amdgcn_ballot_w64(lane < w.S && w.slot[min(lane, w.S - 1)] == slot);
        if (mk >> lane & 1) rows[__popcll(mk & ((1ull << lane) - 1ull))] = lane;
        cnt = __popcll(mk);
    } else {
        const int2 rn = w.run[slot];
        first = rn.x;
        list = w.perm + first;
        cnt = rn.y;
    }
    if (rank <= 16 * rt0) cnt = 0;
    __syncthreads();
    if constexpr (!LIST) {
        const size_t pitch = (size_t)w.S * Rp;
        for (int e = threadIdx.x; e < cnt * 16 * NR; e += 64 * W) {
            const int p = e / (16 * NR), r = e % (16 * NR);
            hl[p][r] = lora_h(h + (size_t)rows[p] * Rp + r, splits, pitch);
        }
        __syncthreads();
    }
    floatx4 acc[NR][4];
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[r][j] = (floatx4){0.f, 0.f, 0.f, 0.f};
    struct Step {
        floatx4 x[4];
        float h[4][NR];
    };
    auto numbers = [&](int p0, int (&rw)[4]) {
#pragma unroll
        for (int u = 0; u < 4; u++) rw[u] = list[min(p0 + 4 * u + kq, cnt - 1)];
    };
    auto load = [&](int p0, const int (&rw)[4], Step &st) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            st.x[u] = row4<true>(x + (size_t)rw[u] * N, c, N);   // (columns past N: not kept)
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const int p = min(p0 + 4 * u + kq, cnt - 1);
                if constexpr (LIST) st.h[u][r] = h[(size_t)(first + p) * Rp + 16 * r + m];
                else st.h[u][r] = hl[p][16 * r + m];
            }
            // (rows past the slot's: zeros on both sides, whatever the clamped row holds)
            const bool live = p0 + 4 * u + kq < cnt;
#pragma unroll
            for (int j = 0; j < 4; j++) st.x[u][j] = live ? st.x[u][j] : 0.0f;
#pragma unroll
            for (int r = 0; r < NR; r++) st.h[u][r] = live ? st.h[u][r] : 0.0f;
        }
    };
    int p0 = 16 * wave;
    if (p0 < cnt) {
        int rw[4];
        Step cur, nxt;
        numbers(p0, rw);
        load(p0, rw, cur);
        numbers(p0 + 16 * W, rw);
        for (; p0 < cnt; p0 += 16 * W) {
            int rn[4];
            numbers(p0 + 32 * W, rn);
            load(p0 + 16 * W, rw, nxt);
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int r = 0; r < NR; r++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        acc[r][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(cur.h[u][r], cur.x[u][j], acc[r][j], 0, 0, 0);
            cur = nxt;
#pragma unroll
            for (int u = 0; u < 4; u++) rw[u] = rn[u];
        }
    }
    for (int r = 0; r < NR; r++) {
        __syncthreads();
        // lane (m, kq): columns 4 m + j, ranks 4 kq + i
#pragma unroll
        for (int q = 0; q < NR; q++)
            if (q == r)
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) red[wave][lane][4 * i + j] = acc[q][j][i];
        __syncthreads();
        for (int e = threadIdx.x; e < 1024; e += 64 * W) {
            const int rk = side1 ? e & 15 : e >> 6, col = side1 ? e >> 4 : e & 63;
            const int ln = (col >> 2) + 16 * (rk >> 2), at = 4 * (rk & 3) + (col & 3);
            float v = red[0][ln][at];
#pragma unroll
            for (int q = 1; q < W; q++) v += red[q][ln][at];
            const int k = 16 * (rt0 + r) + rk;
            // (past the rank: zeros, also where a row of infinities shrank to NaN)
            v = k < rank ? v * meta.scale : 0.0f;
            if (k < max_rank && c0 + col < N)
                out[side1 ? ((size_t)slot * N + c0 + col) * max_rank + k : ((size_t)slot * max_rank + k) * N + c0 + col] = v;
        }
    }
}

template <typename T, bool JOIN>
__global__ __launch_bounds__(256) void coli_lora_expand(LoraRows w, LoraSide<T> s, int Rp) {
    extern __shared__ float hs[];
    lora_expand_block<T, JOIN>(w, s, Rp, blockIdx.x, blockIdx.y, hs);
}
template <typename T, int NR, int W>
__global__ __launch_bounds__(64 * W) void coli_lora_outer(LoraRows w, LoraSide<T> s0, LoraSide<T> s1, int Rp, int max_rank) {
    lora_outer_block<T, NR, W, true>(w, s0, s1, Rp, max_rank, blockIdx.x, blockIdx.y, blockIdx.z != 0);
}
// Up to COLI_LORA_BALLOT rows both run in one launch, the expand's workgroups
// (ne; none without dx) first.
template <typename T, int NR, bool JOIN>
__global__ __launch_bounds__(256) void coli_lora_finish(LoraRows w, LoraSide<T> s0, LoraSide<T> s1, LoraSide<T> e, int Rp,
                                                        int max_rank, int ne, int tiles, int cols) {
    extern __shared__ float hs[];
    const int b = blockIdx.x;
    if (b < ne) {
        lora_expand_block<T, JOIN>(w, e, Rp, b % tiles, b / tiles, hs);
    } else {
        const int o = b - ne, half = (int)(gridDim.x - ne) / 2, r = o % half;
        lora_outer_block<T, NR, 4, false>(w, s0, s1, Rp, max_rank, r % cols, r / cols, o >= half);
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Column splits of one side's shrink; `groups` workgroups without splits, over
// both sides if there are two, `columns` the columns that they take together.
// Up to COLI_LORA_BALLOT rows (four waves) workgroups of at least a step a wave,
// about two a CU. Beyond (eight waves, whose LDS mostly leaves a CU room for
// one): one side by the rounds of workgroups, each with a fixed part of about
// 2900 columns' time (1024 x 14336, rank 64, 69 tiles, the whole call: 1, 2, 3,
// 4, 6, 8 splits 352, 316, 306, 325, 314, 322 us); two sides, whose splits
// differ, as many as fit into one round if that leaves each side some (the
// adapter gradients of 512 x 4096 x 4096, rank 64: 43 us against 49 for two
// rounds' worth), else two rounds' worth (2048 x 4096 x 14336, rank 32: 106
// against 117).
static int shrink_splits(const DevCtx *ctx, int S, long groups, long columns, int N, bool two) {
    const long cus = ctx->cu_count ? ctx->cu_count : 256;
    if (S <= COLI_LORA_BALLOT) {
        const long cols = std::max(256L, columns / (2 * cus));
        return (int)std::max(1L, std::min((N + cols / 2) / cols, two ? 4L : 16L));
    }
    if (two) {
        const long cols = std::max(512L, columns / (2 * groups <= cus ? cus : 2 * cus));
        return (int)std::max(1L, std::min((2 * groups <= cus ? N : N + cols / 2) / cols, 4L));
    }
    long best = 1, least = 0;
    for (long s = 1; s <= 8 && s * 512 <= std::max(512, N); s++) {
        const long t = (groups * s + cus - 1) / cus * (N / s + 2900);
        if (s == 1 || t < least) {
            least = t;
            best = s;
        }
    }
    return (int)best;
}

static int lora_tiles(int S, int slots) {
    return S <= COLI_LORA_BALLOT ? S : S / COLI_LORA_TILE + std::min(S, slots + 1);
}

// Shrink workgroups of one side without splits.
static long lora_groups(int S, const ColiHipLora *l) {
    return (long)lora_tiles(S, l->slots) * (l->Rp >= 64 ? l->Rp / 64 : 1);
}

// The rows' grouping, and (beyond COLI_LORA_BALLOT rows) the launch that makes
// it; what it took along of the operand builds has nblocks 0 afterwards.
static int lora_rows(DevCtx *ctx, const ColiHipLora *l, const int *slot_dev, int S, LoraRows *w, ColiPrepArgs *ride,
                     ColiTPrepArgs *tride) {
    *w = LoraRows{};
    w->slot = slot_dev;
    w->meta = l->meta;
    w->S = S;
    w->slots = l->slots;
    if (S <= COLI_LORA_BALLOT) return 1;
    const size_t nt = (size_t)lora_tiles(S, l->slots);
    const size_t tb = nt * sizeof(int4), rb = (size_t)(l->slots + 1) * sizeof(int2), pb = (size_t)S * sizeof(int);
    if (!reserve_kept(ctx, &ctx->lora_list, tb + rb + pb + 2 * sizeof(int), 0)) return 0;
    uint8_t *p = (uint8_t *)ctx->lora_list.p;
    w->tile = (int4 *)p;
    w->run = (int2 *)(p + tb);
    w->perm = (int *)(p + tb + rb);
    w->ntile = (int *)(p + tb + rb + pb);
    // (a counter for each wave and slot: about 32 KiB of LDS at most)
    const size_t bins = (size_t)l->slots + 1;
    const int rb2 = (ride->nblocks + 1) / 2, rb4 = (ride->nblocks + 3) / 4;
    if (l->slots <= 512) {
        hipLaunchKernelGGL((coli_lora_sort<16>), dim3(1 + (ride->nblocks ? rb4 : tride->nblocks)), dim3(1024),
                           16 * bins * sizeof(int), ctx->stream, *w, *ride, *tride);
        tride->nblocks = 0;
    } else {
        hipLaunchKernelGGL((coli_lora_sort<8>), dim3(1 + rb2), dim3(512), 8 * bins * sizeof(int), ctx->stream, *w, *ride,
                           ColiTPrepArgs{});
    }
    ride->nblocks = 0;
    return hip_check(hipGetLastError(), "adapter rows");
}

template <typename T>
static LoraSide<T> lora_side(const ColiHipLora *l, bool b, const float *x, float *h, float *out, int splits) {
    LoraSide<T> s = {};
    s.x = x;
    s.v = (const T *)(b ? l->bt : l->a);
    s.h = h;
    s.out = out;
    s.N = b ? l->O : l->I;
    s.Np = b ? l->Op : l->Ip;
    s.splits = splits;
    return s;
}

// Up to COLI_LORA_BALLOT rows the launch also runs `ride`; beyond, its
// workgroups have eight waves and the sort has run it.
template <typename T>
static int launch_shrink(DevCtx *ctx, const ColiHipLora *l, const LoraRows &w, const LoraSide<T> &s0,
                         const LoraSide<T> &s1, int sides, const ColiPrepArgs &ride) {
    const int tiles = lora_tiles(w.S, l->slots), nrt = l->Rp / 16, sp = std::max(s0.splits, sides > 1 ? s1.splits : 1);
    const int nr = nrt >= 4 ? 4 : nrt, nz = nrt / nr, nown = tiles * sp * sides * nz;
#define COLI_SHRINK(NR, W)                                                                                        \
    hipLaunchKernelGGL((coli_lora_shrink<T, NR, W>), dim3(nown + ride.nblocks), dim3(64 * W), 0, ctx->stream, w, s0, \
                       s1, l->Rp, nz, tiles, sp, nown, ride)
    if (w.S <= COLI_LORA_BALLOT) {
        if (nr == 1) COLI_SHRINK(1, 4);
        else if (nr == 2) COLI_SHRINK(2, 4);
        else COLI_SHRINK(4, 4);
    } else {
        if (nr == 1) COLI_SHRINK(1, 8);
        else if (nr == 2) COLI_SHRINK(2, 8);
        else COLI_SHRINK(4, 8);
    }
#undef COLI_SHRINK
    return hip_check(hipGetLastError(), "adapter shrink");
}

template <typename T>
static int launch_expand(DevCtx *ctx, const ColiHipLora *l, const LoraRows &w, const LoraSide<T> &s) {
    const dim3 grid(lora_tiles(w.S, l->slots), (s.Np + 511) / 512);
    const size_t shm = (size_t)16 * (l->Rp + 1) * sizeof(float);
    if (s.parts)
        hipLaunchKernelGGL((coli_lora_expand<T, true>), grid, dim3(256), shm, ctx->stream, w, s, l->Rp);
    else
        hipLaunchKernelGGL((coli_lora_expand<T, false>), grid, dim3(256), shm, ctx->stream, w, s, l->Rp);
    return hip_check(hipGetLastError(), "adapter expand");
}

// Up to COLI_LORA_BALLOT rows: adapter gradients and, with e, the expand.
template <typename T>
static int launch_finish(DevCtx *ctx, const ColiHipLora *l, const LoraRows &w, const LoraSide<T> &s0, const LoraSide<T> &s1,
                         const LoraSide<T> *e) {
    const int nrt = l->Rp / 16, cols = (std::max(l->I, l->O) + 63) / 64, nr = nrt >= 4 ? 4 : nrt, ny = l->slots * (nrt / nr);
    const int tiles = lora_tiles(w.S, l->slots), ne = e ? tiles * ((e->Np + 511) / 512) : 0;
    const size_t shm = (size_t)16 * (l->Rp + 1) * sizeof(float);
#define COLI_FINISH(NR, JOIN)                                                                                    \
    hipLaunchKernelGGL((coli_lora_finish<T, NR, JOIN>), dim3(ne + 2 * cols * ny), dim3(256), shm, ctx->stream, w, s0, \
                       s1, e ? *e : s0, l->Rp, l->max_rank, ne, tiles, cols)
#define COLI_FINISH_NR(JOIN)                \
    if (nr == 1) COLI_FINISH(1, JOIN);      \
    else if (nr == 2) COLI_FINISH(2, JOIN); \
    else COLI_FINISH(4, JOIN)
    if (e && e->parts) {
        COLI_FINISH_NR(true);
    } else {
        COLI_FINISH_NR(false);
    }
#undef COLI_FINISH_NR
#undef COLI_FINISH
    return hip_check(hipGetLastError(), "adapter gradients");
}

// Beyond: adapter gradients alone.
template <typename T>
static int launch_outer(DevCtx *ctx, const ColiHipLora *l, const LoraRows &w, const LoraSide<T> &s0, const LoraSide<T> &s1) {
    const int nrt = l->Rp / 16, cols = (std::max(l->I, l->O) + 63) / 64, nr = nrt >= 4 ? 4 : nrt, ny = l->slots * (nrt / nr);
    const long live = (long)((l->I + 63) / 64 + (l->O + 63) / 64) * ny;
#define COLI_OUTER(NR, W)                                                                                            \
    hipLaunchKernelGGL((coli_lora_outer<T, NR, W>), dim3(cols, ny, 2), dim3(64 * W), 0, ctx->stream, w, s0, s1, l->Rp, \
                       l->max_rank)
#define COLI_OUTER_NR(W)               \
    if (nr == 1) COLI_OUTER(1, W);     \
    else if (nr == 2) COLI_OUTER(2, W); \
    else COLI_OUTER(4, W)
    if (live <= (ctx->cu_count ? ctx->cu_count : 256)) {
        COLI_OUTER_NR(16);
    } else {
        COLI_OUTER_NR(4);
    }
#undef COLI_OUTER_NR
#undef COLI_OUTER
    return hip_check(hipGetLastError(), "adapter gradients");
}

template <typename T>
static int lora_forward(DevCtx *ctx, ColiCudaTensor *t, const ColiHipLora *l, float *y, const float *x, int S,
                        const int *slot_dev) {
    LoraRows w;
    const long groups = lora_groups(S, l);
    const int splits = shrink_splits(ctx, S, groups, groups * l->I, l->I, false);
    ColiPrepArgs ride = {};
    ColiTPrepArgs none = {};
    if (!reserve_kept(ctx, &ctx->lora_h, (size_t)splits * S * l->Rp * sizeof(float), 0) ||
        !gemm_prep_beside(ctx, t, x, S, &ride) || !lora_rows(ctx, l, slot_dev, S, &w, &ride, &none))
        return 0;
    float *h = (float *)ctx->lora_h.p;
    const LoraSide<T> a = lora_side<T>(l, false, x, h, nullptr, splits);
    const LoraSide<T> b = lora_side<T>(l, true, nullptr, h, y, splits);
    return launch_shrink<T>(ctx, l, w, a, a, 1, ride) && gemm_prepared(ctx, t, y, x, S) && launch_expand<T>(ctx, l, w, b);
}

template <typename T>
static int lora_backward(DevCtx *ctx, ColiCudaTensor *t, const ColiHipLora *l, const float *x, const float *dy, int S,
                         const int *slot_dev, float *dx, float *da, float *db) {
    LoraRows w;
    const long groups = lora_groups(S, l), columns = groups * (l->I + l->O);
    const int spa = shrink_splits(ctx, S, 2 * groups, columns, l->I, true);
    const int spb = shrink_splits(ctx, S, 2 * groups, columns, l->O, true);
    const bool few = S <= COLI_LORA_BALLOT;
    const size_t hn = (size_t)S * l->Rp;
    GemmTPlan plan = {};
    ColiPrepArgs none = {};
    if (!reserve_kept(ctx, &ctx->lora_h, (spa + spb + (few ? 0 : 2)) * hn * sizeof(float), 0) ||
        (dx && !gemm_t_plan(ctx, t, dy, S, &plan)) || !lora_rows(ctx, l, slot_dev, S, &w, &none, &plan.prep))
        return 0;
    float *h0 = (float *)ctx->lora_h.p, *h1 = h0 + spa * hn;
    LoraSide<T> sa = lora_side<T>(l, false, x, h0, da, spa), sb = lora_side<T>(l, true, dy, h1, db, spb);
    if (!launch_shrink<T>(ctx, l, w, sa, sb, 2, ColiPrepArgs{})) return 0;
    if (!few) {
        LoraJoin j = {{h0, h1}, {h1 + spb * hn, h1 + (spb + 1) * hn}, {spa, spb}, w.perm, S, l->Rp, (int)((hn / 4 + 255) / 256)};
        hipLaunchKernelGGL(coli_lora_join, dim3(2 * j.nblocks), dim3(256), 0, ctx->stream, j);
        if (!hip_check(hipGetLastError(), "adapter rows join")) return 0;
        sa.h = j.to[0];
        sb.h = j.to[1];
        sa.splits = sb.splits = 1;
    }
    // (beyond COLI_LORA_BALLOT rows ahead of the product, which drives the rows out
    // of the caches)
    if (!few && !launch_outer<T>(ctx, l, w, sa, sb)) return 0;
    if (!dx) return !few || launch_finish<T>(ctx, l, w, sa, sb, nullptr);
    LoraSide<T> e = lora_side<T>(l, false, nullptr, sb.h, dx, sb.splits);
    e.sorted = !few;
    if (plan.parts) {   // the expand joins the K splits
        e.part = plan.part;
        e.parts = plan.parts;
    }
    return gemm_t_run(ctx, t, dx, dy, S, plan, !e.parts) &&
           (few ? launch_finish<T>(ctx, l, w, sa, sb, &e) : launch_expand<T>(ctx, l, w, e));
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
    if (!out || I < 4 || O < 4 || I > (1 << 20) || O > (1 << 20) || slots < 1 || slots > COLI_LORA_MAX_SLOTS ||
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
    const size_t yb = (size_t)S * t->O * 4;
    if (!ctx || ranges_overlap(y_dev, yb, x_dev, (size_t)S * t->I * 4) || ranges_overlap(y_dev, yb, slot_dev, (size_t)S * 4))
        return 0;
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
    // the inputs are read until the last launch: no output lies over one, or over another output
    const void *at[6] = {dx_dev, da_dev, db_dev, x_dev, dy_dev, slot_dev};
    const size_t rank = (size_t)l->slots * l->max_rank * 4;
    const size_t n[6] = {(size_t)S * t->I * 4, rank * t->I, rank * t->O, (size_t)S * t->I * 4, (size_t)S * t->O * 4, (size_t)S * 4};
    for (int i = 0; i < 3; i++)
        for (int j = i + 1; j < 6; j++)
            if (at[i] && ranges_overlap(at[i], n[i], at[j], n[j])) return 0;
    forget_emitted(ctx, da_dev, (size_t)l->slots * l->max_rank * l->I * sizeof(float));
    forget_emitted(ctx, db_dev, (size_t)l->slots * l->max_rank * l->O * sizeof(float));
    switch (l->dtype) {
    case 0: return lora_backward<float>(ctx, t, l, x_dev, dy_dev, S, slot_dev, dx_dev, da_dev, db_dev);
    case 1: return lora_backward<_Float16>(ctx, t, l, x_dev, dy_dev, S, slot_dev, dx_dev, da_dev, db_dev);
    default: return lora_backward<bf16_t>(ctx, t, l, x_dev, dy_dev, S, slot_dev, dx_dev, da_dev, db_dev);
    }
}
