/* coli_hip_ext.h -- entry points libcoli_hip.so adds beyond the reference ABI.
 *
 * None of these has a counterpart in c/backend_cuda.h; each states the
 * reference code whose behaviour it provides on the device.
 */
#ifndef COLI_HIP_EXT_H
#define COLI_HIP_EXT_H

#include "coli_backend_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Resident MXFP4 (fmt=7) tensor from its native bytes: q4 [O, ceil(I/2)]
 * e2m1 nibbles, e8 [O, ceil(I/32)] ue8m0 exponents (the layout of
 * c/quant.h:1375-1390). The CUDA backend has no resident fmt=7 group path
 * (c/backend_cuda.cu:1636-1643); this is new capability. */
int coli_hip_tensor_upload_mxfp4(ColiCudaTensor **tensor, const unsigned char *q4,
                                 const unsigned char *e8, int I, int O, int device);

/* Resident MXFP4 tensor from the 16-row interleaved layout of
 * coli_fp4_pack_rows16_v10 (c/deepseek_v4.c:10975-10993): O % 16 == 0,
 * I % 128 == 0. */
int coli_hip_tensor_upload_fp4_rows16(ColiCudaTensor **tensor, const unsigned char *packed_data,
                                      const unsigned char *packed_scales, int I, int O,
                                      int device);

/* Upload whose weight source is already in device memory (row-major source
 * layout, e.g. landed there by a GPU-side loader); scales come from the host:
 * f32 (fmt 2/4) or ue8m0 bytes (fmt 7, e8 != NULL). Same semantics otherwise
 * as coli_cuda_tensor_upload_g. */
int coli_hip_tensor_upload_from_device(ColiCudaTensor **tensor, const void *weights_dev,
                                       const float *scales, const unsigned char *e8, int fmt,
                                       int I, int O, int device, int gs);

/* native_quant contract on the device: every activation row is first
 * quantize-dequantized to e4m3 in blocks of 128 with an e8m0 scale
 * (c/deepseek_v4.c:10495-10520), then multiplied with the resident MXFP4
 * tensor (coli_fp4_matmul_batch_ref, c/deepseek_v4.c:10906-10933; batch 1 is
 * coli_fp4_matvec_ref, 10571-10605). Host pointers; returns 1 / 0. */
int coli_hip_fp4_matmul_qdq(ColiCudaTensor *tensor, float *y, const float *x, int S);

/* Same, device pointers, asynchronous on the backend stream. */
int coli_hip_fp4_matmul_qdq_dev(ColiCudaTensor *tensor, float *y_dev, const float *x_dev, int S);

/* MXFP4 with int8 activations: replaces matmul_mxfp4_i8 (c/quant.h:1441-1515,
 * the K3 IDOT path selected by K3_IDOT=1, c/kimi_k3.c). Each activation row
 * is quantized per 32 columns to int8 (sc = max|x| / 127, q = rint(x / sc)
 * clamped to +-127, bit-exact with the reference) and multiplied with the
 * MXFP4 weights; I % 32 != 0 falls back to the float path as the reference
 * does. Stateless like coli_cuda_matmul_mxfp4 (host q4 [O][I/2], e8
 * [O][I/32]). Returns 1 / 0 (y untouched on failure). */
int coli_hip_matmul_mxfp4_i8(float *y, const float *x, const unsigned char *q4,
                             const unsigned char *e8s, int S, int I, int O);

/* Same on a resident MXFP4 tensor: host pointers (synchronous) / device
 * pointers (asynchronous on the backend stream). */
int coli_hip_fp4_matmul_i8(ColiCudaTensor *tensor, float *y, const float *x, int S);
int coli_hip_fp4_matmul_i8_dev(ColiCudaTensor *tensor, float *y_dev, const float *x_dev, int S);

/* fmt=2 (int4, one f32 scale per row) with int8 activations: replaces the
 * reference's IDOT path for fmt=2 experts (c/colibri.c:937-945: qrow_i8
 * c/quant.h:581-586 per row, then matmul_i4_idot c/quant.h:924-933 with
 * dot_i4i8 674-801). Each row is quantized to int8 (s = max|x| / 127, at least
 * 1e-12; q = rint(x * (1 / s))), the integer dot is exact, and y[s, o] =
 * (float)dot * scale[o] * s: bitwise the reference's result. I <= 16512.
 * Resident fmt=2 tensor; host pointers (synchronous) / device pointers
 * (asynchronous on the backend stream). Returns 1 / 0 (y untouched on
 * failure). */
int coli_hip_matmul_i4_idot(ColiCudaTensor *tensor, float *y, const float *x, int S);
int coli_hip_matmul_i4_idot_dev(ColiCudaTensor *tensor, float *y_dev, const float *x_dev, int S);

/* ---- fused MoE layer (router -> union -> experts -> SwiGLU -> scatter) ---- */
typedef struct ColiHipMoe ColiHipMoe;

typedef struct {
    int D, I, E, K;        /* hidden, expert intermediate, routed experts, top-k */
    int route_mode;        /* 0 softmax then top-k (c/olmoe.c:666-681)
                              1 sigmoid, choice = sigmoid + bias (c/colibri.c:3978-4126)
                              2 sigmoid + bias select, weights renormalized over the
                                selection (c/kimi_k3.c:1337-1356)
                              3 DeepSeek-V4: sqrt(softplus) + bias select, weights
                                score / sum x routed_scale (c/deepseek_v4.c:1368-1432) */
    int norm_topk;
    float topp;            /* 0 disables */
    float routed_scale;    /* 1.0 for none */
    int has_shared;        /* one always-on expert, added after the routed sum */
    float swiglu_limit;    /* > 0: DeepSeek-V4 clamped SwiGLU (c/deepseek_v4.c:1434-1448) */
} ColiHipMoeConfig;

/* Router weights f32 [E, D] (+ bias [E] or NULL) are copied to the device;
 * expert tensors are resident handles of one device (gate/up [I, D], down
 * [D, I]). All experts must share one storage kind. */
int coli_hip_moe_create(ColiHipMoe **moe, int device, const ColiHipMoeConfig *cfg,
                        const float *router_w, const float *router_bias,
                        ColiCudaTensor *const *gates, ColiCudaTensor *const *ups,
                        ColiCudaTensor *const *downs, ColiCudaTensor *shared_gate,
                        ColiCudaTensor *shared_up, ColiCudaTensor *shared_down);
void coli_hip_moe_free(ColiHipMoe *moe);

/* Device-resident forward of S <= 2048 rows (decode, verification or
 * prefill; S * K <= 16384): x_dev [S, D] f32 -> out_dev [S, D] f32,
 * asynchronous on the backend stream (no host sync, no allocation after the
 * first call at a given S; a captured forward stays valid when later ones have
 * more rows). Up to 32 rows the experts run the tiled GEMV,
 * beyond it the grouped GEMM. */
int coli_hip_moe_forward_dev(ColiHipMoe *moe, const float *x_dev, float *out_dev, int S);

/* Host forward with routing read back: idx/w [S, K], keff [S] (may be NULL). */
int coli_hip_moe_forward(ColiHipMoe *moe, const float *x, float *out, int S, int *idx,
                         float *w, int *keff);

/* Union of the last forward: nu and the unique expert ids in first-seen order
 * (c/colibri.c:4146-4152). Synchronizes. */
int coli_hip_moe_last_union(ColiHipMoe *moe, int *nu, int *uniq);

/* coli_cuda_pipe_gemm (device pointers, asynchronous on the backend stream)
 * that allocates nothing. No counterpart in the reference: it is for callers
 * that cannot allocate device memory (code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc). Every buffer beyond x and
 * y lives in one static 8 MiB device array per GPU, held until the process
 * ends. Limits: S <= 16 rows and I <= 16384 (larger calls return 0 with a
 * diagnostic); results are bitwise those of coli_cuda_pipe_gemm. All calls on
 * one GPU share that array: calls that overlap on one GPU (other host
 * threads, other streams) race. Returns 1 / 0. */
int coli_hip_pipe_gemm_noalloc(ColiCudaTensor *tensor, float *y_dev, const float *x_dev, int S);

/* ---- adapters beside a resident projection, and gradients through it --------
 * For serving many fine-tuned variants of one quantized model, and for tuning
 * them: the quantized matrix stays frozen. Device pointers, f32 rows, contiguous;
 * asynchronous on the backend stream (an input written on another stream must
 * be complete or waited for first). Workspaces grow on first use at a size and are
 * shared by the calls of a device, which its one stream orders; a captured
 * graph stays valid when later calls grow them, and must be replayed on that
 * stream. S <= 65535. None of these has a counterpart in the reference. */

/* A bank of low-rank adapters for one projection of width I -> O: slot a holds
 * A [rank, I], B [O, rank] and a scale. dtype of the factors: 0 f32, 1 fp16,
 * 2 bf16. I and O at least 4 (and at most 2^20), slots <= 1024, max_rank <= 256.
 * Slots start empty. */
typedef struct ColiHipLora ColiHipLora;
int coli_hip_lora_create(ColiHipLora **lora, int device, int I, int O, int slots, int max_rank, int dtype);
void coli_hip_lora_free(ColiHipLora *lora);
/* Copy an adapter into its slot (device pointers, row-major, of the bank's
 * dtype; asynchronous: they must hold their values until the copy has run).
 * rank 0 empties the slot; the factors are then not read. */
int coli_hip_lora_set_dev(ColiHipLora *lora, int slot, const void *a_dev, const void *b_dev, int rank, float scale);
/* y[s] = W x[s] + scale_a B_a (A_a x[s]) with a = slot_dev[s]: the projection
 * of coli_cuda_pipe_gemm and each row's adapter in one call. A slot number
 * outside the bank, or of an empty slot: no adapter. y must not overlap x or slot_dev. */
int coli_hip_lora_gemm_dev(ColiCudaTensor *tensor, ColiHipLora *lora, float *y_dev, const float *x_dev, int S,
                           const int *slot_dev);
/* Gradients of that call from dy [S, O]: dx [S, I] (NULL: not wanted), and for
 * every slot of the bank da [slots, max_rank, I] and db [slots, O, max_rank]
 * (written whole: zeros past a slot's rank and where no row has the slot). None
 * of them may overlap an input or another. */
int coli_hip_lora_grad_dev(ColiCudaTensor *tensor, ColiHipLora *lora, const float *x_dev, const float *dy_dev, int S,
                           const int *slot_dev, float *dx_dev, float *da_dev, float *db_dev);
/* Input gradient of coli_cuda_pipe_gemm: dx[S, I] = dy[S, O] W. dx must not
 * overlap dy. The scales of 32 columns are held under the largest of them over
 * all O rows: a weight is off by at most 2^-28 of that scale (MXFP4: 2^-34)
 * beside 2^-20 of itself, so rows of W whose scales lie farther below count as
 * zero. (So too for the dx of coli_hip_lora_grad_dev.)
 * The first call on a tensor also lays out its scales a second time: 190 us with
 * the allocation for 14336 x 4096, as long as the product of 512 rows. They count
 * in the tensor's bytes and the device's statistics from then on, are freed with
 * it and kept current by coli_cuda_tensor_update. That first call (or the first
 * coli_hip_lora_grad_dev with a dx) is refused under capture. */
int coli_hip_gemm_t_dev(ColiCudaTensor *tensor, float *dx_dev, const float *dy_dev, int S);

/* ---- load balance of routed rows -------------------------------------------
 * Per-expert counts and the balance loss of T routed rows by sequence, and the
 * gradient of the router's logits. Device pointers, asynchronous on the
 * device's stream. None has a counterpart in the reference.
 *
 * Sequence i is the rows [offsets[i], offsets[i + 1]) (offsets [n + 1],
 * ascending, int32; NULL with n = 1: all rows); rows whose mask byte is 0 count
 * for nothing (mask [T]; NULL: all count). idx [T, K] are the selected experts,
 * of which the first keff[t] are live (NULL: all K); an index outside 0..E-1 is
 * not counted. p is the router's score of a row divided by its sum: softmax
 * (route_mode 0), sigmoid (1, 2), sqrt-softplus (3), without the selection
 * bias. With c_e the live selections of expert e in the sequence, C their sum
 * and n_i its rows:
 *   counts[i, e] = c_e, rows[i] = n_i,
 *   loss[i] = sum_e (E c_e / C) (1 / n_i) sum_t p[t, e]      (0 where C or n_i is 0)
 * 1.0 is balance (top-K of equal loads). E <= 1024, K <= min(64, E), n <= 16384, T <= 2^24. No
 * output may overlap an input or another output. */
int coli_hip_balance_dev(int device, const float *logits, const int *idx, const int *keff, const unsigned char *mask,
                         const int *offsets, int n, int T, int E, int K, int route_mode, float *loss, int *counts,
                         int *rows);
/* dlogits [T, E] from dloss [n] and the forward's counts and rows (the counts
 * carry no gradient). Masked rows get zeros; rows of no sequence are left as
 * they were. dlogits may be logits, and must not overlap any other input. */
int coli_hip_balance_grad_dev(int device, const float *logits, const unsigned char *mask, const int *offsets, int n,
                              int T, int E, int route_mode, const float *dloss, const int *counts, const int *rows,
                              float *dlogits);
/* coli_hip_balance_dev over the last forward of a MoE layer (its rows, its own
 * router logits, selections and route mode): the one that ran last on the
 * stream before this call, queued by a call or by a graph's replay. mask and
 * offsets are for that forward's rows. Refused before the first forward and
 * after one that failed. */
int coli_hip_moe_last_balance_dev(ColiHipMoe *moe, const unsigned char *mask, const int *offsets, int n, float *loss,
                                  int *counts, int *rows);

/* ---- rows sorted by expert, and back ---------------------------------------
 * What lies between a router and the experts: for experts on other devices
 * (the sorted rows are what is sent), and for tuning through them. Device
 * pointers, contiguous, asynchronous on the device's stream; workspaces and
 * captures as above. No atomics on floating values: the same call gives the same
 * bits. No output may overlap an input or another output. None has a counterpart
 * in the reference.
 *
 * Sort the live selections of T rows by expert: idx [T, K], of which the first
 * keff[t] are live (NULL: all K), none of a row whose mask byte is 0 (NULL: all
 * rows count), nor one outside 0..E-1. Selection s = t K + k; the order is by
 * expert, then by s.
 *   offsets [E + 1]: expert e has the sorted rows [offsets[e], offsets[e + 1])
 *   src [T K]:       the selection of each sorted row
 *   pos [T, K]:      the sorted row of each selection, -1 where it is not live
 *   xs [T K, row_bytes]: the rows, xs[r] = x[src[r] / K], x [T, row_bytes]: of any
 *                    type (x and xs NULL: not wanted)
 * src and xs behind the last live selection are left as they were. Gradient of x:
 * coli_hip_combine_dev of xs's, without weights. T from 0 to 2^23, E <= 1024, K <=
 * 64, T K <= 2^30, rows of up to 64 MiB. */
int coli_hip_dispatch_dev(int device, const int *idx, const int *keff, const unsigned char *mask, int T, int E, int K,
                          const void *x, size_t row_bytes, int *offsets, int *src, int *pos, void *xs);
/* out[t] = sum_k w[t, k] ys[pos[t, k]] over the places pos [T, K] within 0..N-1
 * (others count for nothing, whatever their weight); w [T, K] f32 (NULL: ones), ys
 * [N, D] and out [T, D] of dtype 0 f32, 1 fp16, 2 bf16. Summed in f32 in the order
 * of k, rounded once. Rows of ys that no place names count for nothing. */
int coli_hip_combine_dev(int device, const void *ys, int dtype, const int *pos, const float *w, int T, int K, int N,
                         int D, void *out);
/* Its gradients from dout [T, D]: dys[pos[t, k]] = w[t, k] dout[t] (rows that no
 * place names are left as they were) and dw[t, k] = <dout[t], ys[pos[t, k]]> (0
 * where the place is outside), the product in f32. dys or dw NULL: not wanted (ys may be
 * NULL without dw). No row may be named twice where dys is wanted. */
int coli_hip_combine_grad_dev(int device, const void *ys, int dtype, const int *pos, const float *w, const void *dout,
                              int T, int K, int N, int D, void *dys, float *dw);

/* ---- MXFP4: quantization, and products of 4-bit rows ------------------------
 * Device pointers, asynchronous on the stream, workspaces and captures as above.
 * None has a counterpart in the reference.
 *
 * x [rows, cols] of dtype 0 f32, 1 fp16, 2 bf16 to the native MXFP4 bytes of
 * coli_hip_tensor_upload_mxfp4: q4 [rows, ceil(cols / 2)], e8 [rows, ceil(cols /
 * 32)]. The scale of 32 columns is the smallest power of two, 2^-126 at least, that
 * holds their largest magnitude within 6 (the rule of the e4m3 path: nothing
 * saturates); a block of zeros has scale 1; one with an infinity or NaN has byte
 * 255 and codes 0, which is NaN to whatever reads it. Codes are the nearest, ties to the
 * even code. rows and cols up to 2^24 - 1; without rows nothing is done. */
int coli_hip_mxfp4_quantize_dev(int device, const void *x, int dtype, int rows, int cols, unsigned char *q4,
                                unsigned char *e8);
/* y [rows, cols] from such bytes: code times scale, rounded once to dtype (byte
 * 0 is scale 0, byte 255 infinity, as in the products with f32 rows). */
int coli_hip_mxfp4_dequantize_dev(int device, const unsigned char *q4, const unsigned char *e8, int rows, int cols,
                                  void *y, int dtype);
/* A resident MXFP4 tensor [O, I] quantized from weights on the device (a fresh
 * handle only; synchronous, as the uploads). The weights must be complete. */
int coli_hip_tensor_quantize_mxfp4(ColiCudaTensor **tensor, const void *weights_dev, int dtype, int I, int O, int device);
/* y[S, O] = Q(x) W^T with Q the quantizer above (a row's 32-column blocks) and W a
 * resident MXFP4 tensor, on the fp4 matrix units: exact products, f32 sums. A scale
 * byte of 255 is NaN here, 0 is 2^-127. Host pointers (synchronous) / device pointers
 * (asynchronous; y must not overlap x). S up to 2^23, I up to 2^21, O up to 2^27 - 16. The
 * gradient that passes it (straight through Q) is coli_hip_gemm_t_dev. */
int coli_hip_fp4_matmul_a4(ColiCudaTensor *tensor, float *y, const float *x, int S);
int coli_hip_fp4_matmul_a4_dev(ColiCudaTensor *tensor, float *y_dev, const float *x_dev, int S);
/* The experts' matrices for that product over sorted rows: E <= 1024 resident
 * MXFP4 tensors [O, I] of one shape (I and O as above) on one device; with ups a
 * second one each, and silu(gate) * up as the result (swiglu_limit > 0: the clamped
 * form). The tensors must outlive the set. */
typedef struct ColiHipExperts ColiHipExperts;
int coli_hip_experts_create(ColiHipExperts **experts, int device, int E, ColiCudaTensor *const *gates,
                            ColiCudaTensor *const *ups, float swiglu_limit);
void coli_hip_experts_free(ColiHipExperts *experts);
/* y[r] = W_e Q(x row of r) for the sorted rows offsets[e] <= r < offsets[e + 1] (ascending;
 * taken within 0..N) of y [N, O]; other rows of y are left as they were. The row is
 * x[src[r] / K] with src (of coli_hip_dispatch_dev: the rows need not be copied), x[r]
 * without; x is [rows, I], rows at least 1, a row outside it counts as zeros. N and rows up
 * to 2^23; without sorted rows (N 0) nothing is done. */
int coli_hip_experts_a4_dev(ColiHipExperts *experts, float *y, const float *x, int rows, const int *src, int K,
                            const int *offsets, int N);

/* ---- plumbing for benchmarks and tests ----------------------------------- */
/* coli_cuda_pipe_gemm in two halves, so a timer can bracket the GEMV kernel
 * alone: prep names the activations x_dev[S, I] for the tensor's storage
 * kind (no launch); run launches the GEMV y_dev[S, O]. The first run after a
 * prep also launches the fragment build when its kernel needs fragments (the
 * LDS-ring kernel of up to 32768 activations reads x_dev itself), so x_dev
 * must hold its values until the runs are issued. A run must follow the prep
 * of the same kind of tensor and the same S. */
int coli_hip_gemm_prep_dev(ColiCudaTensor *tensor, const float *x_dev, int S);
int coli_hip_gemm_run_dev(ColiCudaTensor *tensor, float *y_dev, int S);
/* As coli_hip_gemm_run_dev, and the output rows are also written, from the
 * GEMV's epilogue, as the activation fragments of `next` (next->I ==
 * tensor->O, fp16 hi + lo with one exponent per row and 32-column group), so
 * that a following coli_hip_gemm_prep_dev(next, y_dev, S) + run needs no
 * fragment build (an FFN's up projection feeding its down projection).
 * Emitted only where it pays and the launch allows it (2..16 rows whose f32
 * form next's GEMV would not convert itself, tensor->O a multiple of 128, a
 * plain launch with an even number of row tiles per wave and no K split);
 * otherwise the later prep builds the fragments as usual. The caller must not
 * modify y_dev between this call and that prep's run; another run writing
 * y_dev drops the emitted fragments. Returns 2 when the fragments were
 * emitted, 1 when only the GEMV ran, 0 on failure. */
int coli_hip_gemm_run_dev_emit(ColiCudaTensor *tensor, float *y_dev, int S, const ColiCudaTensor *next);
/* Fill n bytes of device memory with uniform pseudo-random bytes (seeded,
 * deterministic): synthetic weights for benchmarks without a host round trip. */
int coli_hip_fill_random_u8(int device, void *dev, size_t n, unsigned long long seed);
/* Queue a plain streaming read of `bytes` (a multiple of 16, 16-byte aligned)
 * of device memory on the device's stream: no arithmetic, nothing written.
 * The benchmark's reference for what one launch of a given size can read. */
int coli_hip_stream_read(int device, const void *dev, size_t bytes);
/* The hipStream_t every asynchronous entry point of `device` runs on. */
void *coli_hip_stream(int device);
/* Bytes the tensor streams per full GEMV (weights + scales, tiled storage). */
size_t coli_hip_tensor_stream_bytes(const ColiCudaTensor *tensor);
/* Storage kind: 0 int4+fp16 scales, 1 int4+f32 scales, 2 MXFP4, 3 generic int4. */
int coli_hip_tensor_kind(const ColiCudaTensor *tensor);

#ifdef __cplusplus
}
#endif

#endif
