/* KERNIX-B200 kernel-level C ABI: the sm_100a CUDA kernels behind the model runtime.
 *
 * Plain device pointers, sizes and a cudaStream_t passed as void*; no CUDA or torch types. All matrices
 * are row-major with an explicit leading dimension (elements). Every function returns 0 when the launch
 * was accepted and -1 on bad arguments or a launch error. Kernels whose waits are bounded OR
 * KX_STATUS_TIMEOUT into *status (device memory, may be NULL) instead of hanging; bits that are there stay.
 * Each entry names the reference computation it replaces (KERNIX reference file:line).
 */
#ifndef KX_KERNELS_H
#define KX_KERNELS_H

#include <stddef.h>
#include <stdint.h>

#include "kernix.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KX_STATUS_OK 0
#define KX_STATUS_TIMEOUT 1

/* ---- int8 path (include/kernix_model.h:99-182 kernix_qmatmul) ---- */

/* Per-row dynamic int8 quantisation (kernix_qmatmul :110-142): m = max|x| over the row (NaN wins),
 * sx = m > 0 ? m / 127 : 1, xq = clamp(rint(x * (1/sx)), -127, 127); rows whose m is NaN/inf get sx = NaN
 * (their GEMM output becomes NaN, as the reference's NaN rows). xq columns k..ldq-1 are zeroed. */
KERNIX_API int kx_quant_rows(const float* x, int ldx, int rows, int k, int8_t* xq, int ldq, float* sx, void* stream);

/* kx_quant_rows that also clears zero[0 .. zero_words) once the kernel before it has completed: the row maxima
 * and counters of the kx_gemm_i8_q launch that follows (an internal step of the model runtime). */
KERNIX_API int kx_quant_rows_z(const float* x, int ldx, int rows, int k, int8_t* xq, int ldq, float* sx, uint32_t* zero,
                               int zero_words, void* stream);

/* y = act(((float)acc * sx[row]) * scale[col] + bias[col]) with acc = sum_t xq[row][t] * wq[col][t] in int32
 * on tcgen05 kind::i8 (kernix_qmatmul :143-177 and the step's activation :1854-1856). wq: n x ldw int8,
 * K-major (see kx_prep_i8_weight). ldq, ldw multiples of 16. bias may be NULL (adds 0). */
KERNIX_API int kx_gemm_i8(const int8_t* xq, int ldq, const float* sx, const int8_t* wq, int ldw, const float* scale,
               const float* bias, float* y, int ldy, int m, int n, int k, int act, float alpha, int* status, void* stream);

/* A hidden int8 layer whose output feeds only the next int8 layer (kernix_qmatmul :99-182 twice, :1854-1856):
 * the int8 GEMM of kx_gemm_i8 whose epilogue quantises its own output rows for the next layer, as kx_quant_rows
 * would from y, and writes q_out (m x ldq_out int8; ldq_out >= n, a multiple of 16; columns n .. ldq_out-1 zero;
 * 16-byte aligned) and sx_out (m floats) instead of y: bit for bit the kx_quant_rows result of y. ctl: m + ceil(m/128)
 * words of device memory that must be zero at launch (row maxima and row-group counters); the launch clears
 * zero_next[0 .. zero_words) for the next one. n > 128 (CTA-pair tiles) and at most as many 256-column tiles as
 * CTA pairs resident at once, else -1. */
KERNIX_API int kx_gemm_i8_q(const int8_t* xq, int ldq, const float* sx, const int8_t* wq, int ldw, const float* scale,
                            const float* bias, int m, int n, int k, int act, float alpha, int8_t* q_out, int ldq_out,
                            float* sx_out, uint32_t* ctl, uint32_t* zero_next, int zero_words, int* status, void* stream);

/* A chain of n_layers (2..4) int8 LINEAR steps (kernix_qmatmul :99-182 plus the activation :1854-1856, step after
 * step, each hidden output quantised as the next step's input as kx_quant_rows would) in ONE persistent launch of the
 * CTA-pair int8 GEMM, every layer's tiles in one walk: a tile of layer l > 0 starts once the rows it reads are
 * quantised. a[0] / sx[0]: the chain input quantised (kx_quant_rows_z); a[l] / sx[l] = sx_out[l-1] for l > 0: the
 * buffers layer l-1 writes (m x lda[l] int8, 16-byte aligned; m floats). y: m x n[last] fp32. ctl: (n_layers - 1) x
 * (m + 2 * ceil(m / 128)) words, zero at launch (clear them with the quantiser before). Every n[l] > 128, at most 64
 * tiles of 256 columns per layer, hidden layers of one activation class (ReLU, GELU, none or another); else -1.
 * Bit for bit the results of running the steps one by one. */
KERNIX_API int kx_i8_chain(int n_layers, int m, const int8_t* const* a, const int* lda, const float* const* sx,
                           const int8_t* const* wq, const int* ldw, const float* const* scale, const float* const* bias,
                           const int* k, const int* n, const int* act, const float* alpha, float* const* sx_out,
                           uint32_t* ctl, float* y, int* status, void* stream);

/* One int8 LINEAR step from fp32 activations, the whole of kernix_qmatmul plus the step's activation
 * (include/kernix_model.h:99-182, :1854-1856): quantise x's rows into xq_scratch (rows x ldq int8, ldq =
 * k rounded up to 16) and sx_scratch (rows floats), then y = act(((float)acc * sx) * scale + bias) with the
 * int8 tcgen05 GEMM. The two scratch buffers are device memory supplied by the caller. */
KERNIX_API int kx_linear_i8(const float* x, int ldx, int rows, int k, const int8_t* wq, int ldw, const float* scale,
                            const float* bias, float* y, int ldy, int n, int act, float alpha, int8_t* xq_scratch,
                            float* sx_scratch, int* status, void* stream);

/* kx_linear_i8 for callers that cannot allocate device memory (latency-critical code that cannot take cudaMalloc's
 * device-wide synchronisation, or hosts whose allocator forbids extra device allocations). No counterpart in the
 * reference. Same arguments and result as kx_linear_i8 minus the two scratch buffers: they come from one
 * KX_NOALLOC_SCRATCH_BYTES array compiled into the library (held on every GPU that loads it until exit), so
 * rows * (k rounded up to 16) + 4 * rows (+ alignment) must fit, else it returns -1 with a message. The first call on
 * a device (per CUDA context) loads the module that holds the array, which reserves its 16 MiB there, and looks
 * the array up (cudaGetSymbolAddress): make that call in initialisation code, before any stream capture. Later
 * calls in the same context allocate nothing; after cudaDeviceReset the next call looks the array up again.
 * Calls share the array: calls whose work overlaps on the GPU race, so order them on one stream. */
#define KX_NOALLOC_SCRATCH_BYTES (16 << 20)
KERNIX_API int kx_linear_i8_noalloc(const float* x, int ldx, int rows, int k, const int8_t* wq, int ldw, const float* scale,
                                    const float* bias, float* y, int ldy, int n, int act, float alpha, int* status,
                                    void* stream);

/* Failure-detection check of the bounded waits every tcgen05 kernel here uses (the counterpart of the reference's
 * command-buffer error handling, src/kernix_metal.m:259-263, which turns a failed GPU command into -1): one warp
 * waits on an mbarrier with the library's wait helper and a limit of limit_ns (at most 2 s). arrive = 1: the
 * barrier completes and *status is left as it was; arrive = 0: nothing arrives, the wait gives up after limit_ns
 * and ORs KX_STATUS_TIMEOUT (1) into *status, and the launch ends normally. *waited_ns: time spent waiting.
 * Device pointers; returns -1 on bad arguments or a launch error. */
KERNIX_API int kx_probe_bounded_wait(int arrive, unsigned long long limit_ns, int* status, unsigned long long* waited_ns,
                                     void* stream);

/* Small-batch int8 layers with the reduction split over the SMs. kx_i8_split_blocks: K blocks (of 128) per range for an
 * m x n x k layer so that its output tiles times its ranges about fill the SMs (at most KX_I8_SPLIT_MAX ranges).
 * kx_gemm_i8_split_acc: the int32 sums of each K range into plane z of part (ceil(ceil(k / 128) / kbs) planes of
 * m x n int32). kx_i8_rows: one row per block adds the planes (exactly), then ((float)acc * sx) * scale + bias and the
 * activation as the int8 GEMM epilogue does, and stores the fp32 row (q == NULL) or quantises it for the next int8
 * layer exactly as the quantised-output epilogue does (q: m x ldq int8, columns n .. ldq - 1 written 0; sx_out: row
 * scales). n, ldq <= 8192. Bit for bit the results of kx_gemm_i8 / kx_gemm_i8_q (the per-step kernels the
 * reference's kernix_qmatmul :99-182 maps to). */
#define KX_I8_SPLIT_MAX 64
KERNIX_API int kx_i8_split_blocks(int m, int n, int k);
KERNIX_API int kx_gemm_i8_split_acc(const int8_t* xq, int ldq, const int8_t* wq, int ldw, int m, int n, int k, int kbs,
                                   int32_t* part, int* status, void* stream);
KERNIX_API int kx_i8_rows(const int32_t* part, int planes, int m, int n, const float* sx, const float* scale, const float* bias,
                          int act, float alpha, float* y, int ldy, int8_t* q, int ldq, float* sx_out, void* stream);

/* int32 accumulators only (acc[row][col], leading dimension ldacc): exposes the integer result for tests. */
KERNIX_API int kx_gemm_i8_acc(const int8_t* xq, int ldq, const int8_t* wq, int ldw, int32_t* acc, int ldacc, int m, int n, int k,
                   int* status, void* stream);

/* Load-time repack of an I8_COL weight block (the file's k x n, in x out) into n x ldw K-major, zero padded
 * (replaces kernix_qweight_pack :62-81, whose layout served NEON sdot). */
KERNIX_API int kx_prep_i8_weight(const int8_t* q_kn, int k, int n, int8_t* wq, int ldw, void* stream);

/* ---- fp32 dense path (kernix_dense :544-550 -> kernix_matmul_ep_into include/kernix.h:955-976,
 *      src/kernix_metal.m:161-265 MPS+AMX split with the bias_act epilogue :269-299) ---- */

/* y = act(x . W + bias) in 3xTF32 on tcgen05 kind::tf32, fp32 accumulation in TMEM. W is given as the
 * tf32 split planes w_hi, w_lo (n x ldw, K-major, ldw % 4 == 0; see kx_prep_f32_weight). bias may be NULL. */
KERNIX_API int kx_gemm_f32(const float* x, int ldx, const float* w_hi, const float* w_lo, int ldw, const float* bias, float* y,
                int ldy, int m, int n, int k, int act, float alpha, int* status, void* stream);

/* y = act(x . W + bias) + res (ldr >= n): a LINEAR step and the elementwise ADD that consumes it in one kernel
 * (kernix_dense :544-550 followed by kernix_binary_run :877-906), each output written once. The add is the ADD
 * step's round-to-nearest fp32 add on the activation's output, so results are bitwise those of the two steps run
 * apart. y may be res (in place); neither may overlap x. */
KERNIX_API int kx_gemm_f32_res(const float* x, int ldx, const float* w_hi, const float* w_lo, int ldw, const float* bias, float* y,
                    int ldy, int m, int n, int k, int act, float alpha, const float* res, int ldr, int* status, void* stream);

/* kx_gemm_f32 for at most 128 rows with the reduction split into `splits` (<= KX_SPLITK_MAX) ranges of K (multiples
 * of 256) run by separate CTAs -- for layers whose few output tiles would leave most SMs idle (a column-sharded wide
 * layer at small batch) -- then y = act(P[0] + ... + P[splits-1] + bias) added in range order (kx_add_planes).
 * part: splits x m x n floats of device scratch. splits = 1 is kx_gemm_f32 (any m; part unused). */
#define KX_SPLITK_MAX 4
KERNIX_API int kx_gemm_f32_split(const float* x, int ldx, const float* w_hi, const float* w_lo, int ldw, const float* bias,
                                 float* y, int ldy, int m, int n, int k, int act, float alpha, int splits, float* part,
                                 int* status, void* stream);
/* the split count kx_gemm_f32_split should be given for an m x n x k layer: 1 (no split) unless m <= 128, k >= 2048 and
 * the layer's output tiles fill fewer than half the SMs; at most KX_SPLITK_MAX, ranges of at least 1024 */
KERNIX_API int kx_gemm_f32_splits(int m, int n, int k);
KERNIX_API int kx_add_planes(const float* part, int planes, int m, int n, const float* bias, int act, float alpha, float* y,
                             int ldy, void* stream);

/* Load-time transpose + split of a float weight (k x n, in x out) into n x ldw K-major planes
 * hi = tf32(w), lo = w - hi (exact), zero padded. */
KERNIX_API int kx_prep_f32_weight(const float* w_kn, int k, int n, float* w_hi, float* w_lo, int ldw, void* stream);

/* A chain of small fp32 dense layers y_l = act_l(y_{l-1} . W_l + b_l) (kernix_dense :544-550 step after step, each
 * reading only the previous output) and, if softmax, a row softmax of the last (floats_softmax_into
 * include/kernix.h:652-657; then the last layer has at most 64 outputs), in ONE cooperative launch: each layer a phase
 * of CUDA-core tiles over K ranges, partial sums in scratch, added in a fixed order by the next layer (the last
 * layer's by a final phase, which also runs a narrow last layer per row), a bounded grid barrier after each phase;
 * each layer's K ranges depend on its k and n only, so a row's result does not depend on the batch it is in. For batches whose tensor-core GEMMs are dominated by per-launch costs (rows <=
 * KX_MLP_MAX_ROWS). w[l]: k[l] x n[l] row-major fp32; bias[l] may be NULL; ldx and every n[l] but the last multiples of
 * 4, x and scratch 16-byte aligned; scratch: kx_mlp_chain_scratch_floats(m, k, n, n_layers) floats; bar: two words
 * (arrivals at the current grid barrier, barrier generation), zero before the first launch, kept between launches
 * (reset them after a timeout). */
#define KX_MLP_MAX_LAYERS 8
#define KX_MLP_MAX_SPLIT 8
#define KX_MLP_MAX_ROWS 512
KERNIX_API int kx_mlp_chain(const float* x, int ldx, int m, int n_layers, const float* const* w, const float* const* bias,
                            const int* k, const int* n, const int* act, const float* alpha, int softmax, float* y,
                            float* scratch, uint32_t* bar, int* status, void* stream);
KERNIX_API size_t kx_mlp_chain_scratch_floats(int m, const int* k, const int* n, int n_layers);

/* ---- elementwise / row ops (memory-bound) ---- */

/* y[r][c] = act(x[r][c] + bias[c]) (kernix_bias_act :528-541; ACT step :1864-1866). x == y allowed; bias may be NULL. */
KERNIX_API int kx_bias_act(const float* x, float* y, long rows, int cols, const float* bias, int act, float alpha, void* stream);

/* row softmax (floats_softmax_into include/kernix.h:652-657); x == y allowed */
KERNIX_API int kx_softmax_rows(const float* x, float* y, long rows, int cols, void* stream);

/* row layer norm, biased variance, (x-mean)*rstd*gamma + beta (kernix_layer_norm_rows_into include/kernix.h:667-677);
 * gamma/beta may be NULL; x == y allowed */
KERNIX_API int kx_layernorm_rows(const float* x, float* y, long rows, int cols, const float* gamma, const float* beta, float eps,
                      void* stream);

/* y = x * g[c] + b[c] per row (AFFINE step :1882-1890); x == y allowed */
KERNIX_API int kx_affine_rows(const float* x, float* y, long rows, int cols, const float* g, const float* b, void* stream);

/* y[s][i] = x[s][i] + cst[i] per sample of `per` floats (ADD_CONST step :1891-1895); x == y allowed */
KERNIX_API int kx_add_const(const float* x, float* y, long samples, long per, const float* cst, void* stream);

/* elementwise op with size-1 row/column broadcast inside each sample (kernix_binary_run :877-906).
 * a: samples x ra x ca, b: samples x rb x cb, y: samples x R x C; y may alias a or b when shapes match. */
KERNIX_API int kx_binary(const float* a, int ra, int ca, const float* b, int rb, int cb, float* y, long samples, int R, int C, int op,
              void* stream);

/* max / avg k x k pooling, NHWC (kernix_pooling_run :773-807) */
KERNIX_API int kx_pool2d(const float* x, float* y, int B, int H, int W, int C, int Ho, int Wo, int kh, int kw, int sh, int sw, int pt,
              int pl, int type, int count_pad, void* stream);

/* per-sample max / mean over R rows (kernix_global_pool_run :810-830) */
KERNIX_API int kx_global_pool(const float* x, float* y, long B, int R, int C, int type, void* stream);

/* per-sample axis permutation, output axis k = input axis perm[k] (kernix_permute_run :833-862) */
KERNIX_API int kx_permute(const float* x, float* y, long B, int nd, const int* dims, const int* perm, void* stream);

/* copy `cols` columns of each row from x (leading dimension ldx) into y at column offset yoff (leading dimension ldy):
 * CONCAT on the channel axis (:908-921) and SELECT on the last axis (:944-947) */
KERNIX_API int kx_copy_cols(const float* x, long ldx, float* y, long ldy, long yoff, long rows, long cols, void* stream);

/* zero-pad H and W of an NHWC image (kernix_pad_run :949-966) */
KERNIX_API int kx_pad2d(const float* x, float* y, int B, int H, int W, int C, int Ho, int Wo, int pt, int pl, void* stream);

/* nearest upsampling (kernix_upsample_run :968-983) */
KERNIX_API int kx_upsample2d(const float* x, float* y, int B, int H, int W, int C, int Ho, int Wo, int sh, int sw, void* stream);

/* table rows for float ids, NaN rows for ids out of range or not integral (kernix_embedding_run :986-1000) */
KERNIX_API int kx_embedding(const float* ids, long n, const float* table, int vocab, int dim, float* y, void* stream);

/* depthwise conv (groups == cin): out = bias, += x * w per in-range tap, then act (kernix_conv_run :724-752) */
KERNIX_API int kx_conv_depthwise(const float* x, const float* w, const float* bias, float* y, int B, int H, int W, int C, int Co,
                      int Ho, int Wo, int kh, int kw, int sh, int sw, int dh, int dw, int pt, int pl, int act, float alpha,
                      void* stream);

/* Implicit-GEMM convolution (NHWC, weights (ky,kx,ci) x cout as the file stores them) on tcgen05 3xTF32 with
 * fused bias + act; the im2col rows are gathered straight into shared memory, never materialised
 * (replaces kernix_conv_run's im2col + sgemm tiles :662-771). w_hi/w_lo: cout x ldw split planes of the
 * weight (kx_prep_f32_weight), ldw >= kh*kw*cin/groups. Output group g writes channels [g*cog, (g+1)*cog). */
KERNIX_API int kx_conv_f32(const float* x, const float* w_hi, const float* w_lo, int ldw, const float* bias, float* y, int B, int H,
                int W, int C, int Co, int Ho, int Wo, int kh, int kw, int sh, int sw, int dh, int dw, int pt, int pl,
                int groups, int act, float alpha, int* status, void* stream);

/* kx_conv_f32 with caller scratch ws of ws_floats floats (16-byte aligned): when the convolution has stride 1, a
 * multiple of 32 input channels and at most 128 output channels per group, K <= 2048, and output images whose
 * pixels cut into 256-pixel tiles of whole rows or whole images, x is split once into tf32 hi / lo planes in ws
 * (2 * B*H*W*C floats) and the pixel operand is loaded by the TMA as 4-D boxes (zero fill = padding) instead of
 * being gathered by threads; otherwise, or with too little scratch, it is kx_conv_f32. Same results within the
 * 3xTF32 bound (the same products in another order). Same role as kx_conv_f32 (kernix_conv_run :662-771). */
KERNIX_API int kx_conv_f32_ws(const float* x, const float* w_hi, const float* w_lo, int ldw, const float* bias, float* y, int B,
                   int H, int W, int C, int Co, int Ho, int Wo, int kh, int kw, int sh, int sw, int dh, int dw, int pt, int pl,
                   int groups, int act, float alpha, float* ws, size_t ws_floats, int* status, void* stream);

/* scaled dot-product attention per (sample, head): ctx = softmax(scale * Q K^T [+ causal -inf]) V with
 * scale = 1/sqrt(dk) (kernix_attention_run :1015-1046). q: (B*Rq) rows of H*dk at leading dim ldq, k: (B*S) rows
 * of H*dk (ldk), v: (B*S) rows of H*dv (ldv), ctx: (B*Rq) rows of H*dv (ldc). Rq, S <= 128 with head dims <= 64
 * run on the tensor cores (3xTF32), the rest on the CUDA cores. status: device word that receives
 * KX_STATUS_TIMEOUT if a bounded wait gives up (may be NULL). */
KERNIX_API int kx_attention(const float* q, int ldq, const float* k, int ldk, const float* v, int ldv, float* ctx, int ldc, int B,
                 int Rq, int S, int H, int dk, int dv, int causal, int* status, void* stream);

/* ---- paged key-value cache: its pages, the attention of one new token over it, windowed prompt attention ----
 * Extensions next to the ATTENTION step's kx_attention (kernix_attention_run :1005-1048); the reference has no cache.
 *
 * A kx_kv describes a cache in device memory that the caller owns; the struct itself is host memory, read during the
 * call only. K and V live in pools of pages: page p of layer l holds `page` tokens of every key-value head,
 *   K: k + l * k_layer + p * k_page (elements), heads x page x dk, dense;  V: likewise with dv.
 * Sequence slot s holds lens[s] tokens on the pages table[s * max_pages + j], j < ceil(lens[s] / page); the entries
 * behind them are -1. refs[p] counts the table entries that name page p; 0 means free. The tables serve every layer.
 * An empty cache has lens = 0, refs = 0, table = -1; the entry points below keep these consistent.
 * Requirements, else -1: page a power of two up to 1024; dk * size and dv * size multiples of 16 bytes, dk, dv <= 1024;
 * k, v and all strides * size multiples of 16 bytes; pages (and layers) that do not overlap;
 * max_pages * page < 2^31, max_pages < 2^31 - 1024; n_pages, n_seqs <= 2^30; heads * page * dk and heads * page * dv <= 2^28. Calls that change a cache are ordered on one
 * stream (or by events) with those that use it.
 *
 * Requests live in device memory, so a kernel checks them: what it refuses it leaves out, memory-safely, and ORs a bit
 * into *status (device word, may be NULL; never cleared here): KX_STATUS_NO_PAGES, too few free pages or a full table
 * row; KX_STATUS_BAD_REQUEST, a slot, length or page id out of range, or a slot that may not be used so. */
#define KX_KV_F32 0
#define KX_KV_F16 1
#define KX_KV_BF16 2
#define KX_STATUS_NO_PAGES 2
#define KX_STATUS_BAD_REQUEST 4
typedef struct {
    int type;                            /* element type of the pools: KX_KV_F32, KX_KV_F16 or KX_KV_BF16 */
    int layers, n_pages, page, heads, dk, dv;
    int n_seqs, max_pages;               /* slots; pages per slot at most */
    void* k;
    void* v;
    long k_page, k_layer;                /* elements from one page to the next, from one layer to the next */
    long v_page, v_layer;
    int32_t* table;                      /* n_seqs x max_pages */
    int32_t* lens;                       /* n_seqs */
    int32_t* refs;                       /* n_pages */
} kx_kv;

/* bytes of device workspace (16-byte aligned) for extend, fork and compact on this cache; its contents need no
 * preparation and carry nothing from call to call, so calls may share one workspace unless they overlap on the GPU
 * (calls on different streams and concurrently replayed graphs each need their own). 0 if the description is invalid. */
KERNIX_API size_t kx_kv_ws(const kx_kv* c);

/* Room for want[s] more tokens in every slot s (want: n_seqs words; <= 0 asks for nothing): pages are taken for them, lens[s] += want[s]
 * and granted[s] = want[s]; a refused slot is left as it was with granted[s] = 0 (want and granted may be the same
 * array). Slots are served in order and pages taken lowest id first; once a slot's need exceeds what is free, it and
 * every later slot that needs a page is refused. The new tokens are then written by kx_kv_append, layer by layer. */
KERNIX_API int kx_kv_extend(const kx_kv* c, const int32_t* want, int32_t* granted, void* ws, size_t ws_bytes, int* status,
                            void* stream);

/* The last count[s] tokens of every slot s (positions lens[s] - count[s] .. lens[s] - 1) of one layer from fp32 rows
 * s * rows + i, i < count[s] (<= rows; <= 0: none): heads * dk floats of k at leading dimension ldk, heads * dv of v at
 * ldv, rounded to the cache's type (to nearest even). Rows i >= count[s] are not read. k and v must not overlap the pools. The
 * tokens' pages are the slot's alone (append before a fork shares them): what lands in a shared page is there for all of its
 * sequences, and of two slots that write the same token of it in one call either's row stays. */
KERNIX_API int kx_kv_append(const kx_kv* c, int layer, const float* k, int ldk, const float* v, int ldv, const int32_t* count,
                            int rows, int* status, void* stream);

/* dst[i] becomes a copy of the sequence in src[i], i < n <= n_seqs: full pages are shared (refs + 1), a partly filled
 * last page is copied to a fresh page (every layer; lowest free ids, in order of i), so that either may grow. All pairs
 * see the state before the call. Refused: dst[i] not empty (lens != 0), equal to src[i] or already named by an earlier
 * pair, slots or lengths out of range; and, once pages run out, each pair from there on that needs one. A pair with
 * dst[i] < 0 is skipped. A parent's page id out of range is passed on as -1 (and reported). */
KERNIX_API int kx_kv_fork(const kx_kv* c, const int32_t* src, const int32_t* dst, int n, void* ws, size_t ws_bytes, int* status,
                          void* stream);

/* The slots seqs[i], i < n, become empty; each of their pages loses a reference. Slots < 0 are skipped, a slot may be
 * named twice. */
KERNIX_API int kx_kv_free(const kx_kv* c, const int32_t* seqs, int n, int* status, void* stream);

/* Moves pages so that the live ones (refs != 0) are the pages 0 .. *n_live - 1: the r-th free page below n_live takes
 * the contents (every layer), references and table entries of the r-th live page from n_live on. n_live: device word. */
KERNIX_API int kx_kv_compact(const kx_kv* c, int32_t* n_live, void* ws, size_t ws_bytes, void* stream);

/* Attention of one new token per row over the cache (scaled dot products as kx_attention, keys and values read from their
 * pages): row i, i < n, is the last token (position lens - 1, appended before) of slot seqs[i] (seqs NULL: slot i), its H
 * query heads in q + i * ldq (H * dk floats); query head h reads key-value head h / (H / heads). It sees key j when window
 * <= 0, or j > lens - 1 - window, or j < sinks. ctx + i * ldc receives H * dv floats. scale 0 means 1/sqrt(dk); |scale| <
 * 2.3e38. A row with seqs[i] < 0 is left as it was, one whose slot holds no tokens becomes 0, and one whose slot, length or
 * (visible) pages are out of range becomes NaN and is reported. Keys and values that are not seen do not affect results,
 * whatever they hold; q and those that are have to be finite and, q and an fp32 cache, below 2^127 (a head that sees an
 * infinite key becomes NaN, a column with an infinite value NaN). H a multiple of heads, dk, dv <= 128. q and ctx must not
 * overlap each other or the cache. Accuracy is fp32's; against an f16 cache q keeps 2^-22 of itself, or 2^-38 of its head's
 * largest element where that is more, and a weight 2^-22 of itself or 2^-38 of the largest among its 16 keys (positions 16 i
 * to 16 i + 15). ws: kx_attention_paged_ws bytes of device workspace (0: the arguments are invalid), to be shared under
 * kx_kv_ws's rules. Results do not depend on timing: the same call on the same contents gives the same bits. */
KERNIX_API size_t kx_attention_paged_ws(const kx_kv* c, int H, int n);
KERNIX_API int kx_attention_paged(const kx_kv* c, int layer, const float* q, int ldq, int H, const int32_t* seqs, int n, int window,
                                  int sinks, float scale, float* ctx, int ldc, void* ws, size_t ws_bytes, int* status,
                                  void* stream);

/* Attention of prompts with a sliding window whose first tokens stay visible (fp32 rows as kx_attention's, but heads that
 * share keys and values, ragged samples, any length). Sample b has q_len[b] <= Rq query rows b * Rq + i (ldq, H * dk floats)
 * and k_len[b] <= S key and value rows b * S + j (ldk, Hkv * dk; ldv, Hkv * dv); q_len, k_len: device words, NULL = Rq, S.
 * Its queries are the last tokens: query i is at position t = k_len - q_len + i and sees key j when j <= t and (window <= 0
 * or j > t - window or j < sinks). ctx rows b * Rq + i (ldc, H * dv floats); a row that sees nothing (t < 0) becomes 0, rows
 * i >= q_len are left as they were; a sample whose lengths are out of range is reported (KX_STATUS_BAD_REQUEST) and its Rq
 * rows become NaN. Query head h reads key-value head h / (H / Hkv). scale 0 means 1/sqrt(dk); |scale| < 2.3e38. dk, dv <=
 * 128, H a multiple of Hkv. q, k, v must not overlap ctx or ws. ws: kx_attention_window_ws bytes of device workspace (0: the
 * arguments are invalid), 128-byte aligned, shared under kx_kv_ws's rules. Key and value rows that no query of the sample
 * sees do not affect results, not in their last bits either, whatever they hold; a row that some queries see takes part in
 * the roundings of its 64 neighbours. Accuracy is fp32's: products keep 2^-22 of their operands, where an element of q (k or
 * v) is not below 2^-16 of the largest in its row (in its 64 rows), or a weight not below 2^-16 of the largest that its row
 * has among those 64 keys; below that they keep 2^-38 of that largest. Blocks of 128 rows that see NaN, infinities,
 * magnitudes of 2^40 and more, rows of k or v 2^14 times above one of their neighbours, or 64 rows of v all below 2^-40, are
 * computed by plain fp32 code, 8 (128 keys a row) to 300 times slower (2500 keys). */
KERNIX_API size_t kx_attention_window_ws(int B, int S, int Hkv, int dk, int dv);
KERNIX_API int kx_attention_window(const float* q, int ldq, const float* k, int ldk, const float* v, int ldv, float* ctx, int ldc,
                                   int B, int Rq, int S, int H, int Hkv, int dk, int dv, const int32_t* q_len, const int32_t* k_len,
                                   int window, int sinks, float scale, void* ws, size_t ws_bytes, int* status, void* stream);

/* y = max(a*x + b, 0), fused multiply-add then max (src/kernix_metal.m:331-338; include/kernix.h:990) */
KERNIX_API int kx_fma_relu(const float* a, const float* x, const float* b, float* y, size_t n, void* stream);

/* Re-interleave an all-gathered column-sharded output: src = [world][rows][slice] -> y rows x (world * slice)
 * with row pitch ldy: y[r][g * slice + j] = src[(g * rows + r) * slice + j]. (Extension; the reference has no
 * sharding.) */
KERNIX_API int kx_unshard_cols(const float* src, int world, long rows, int slice, float* y, int ldy, void* stream);

/* One time step of one direction of an LSTM (kind 0), GRU (1) or SimpleRNN (2) (kernix_rnn_dir,
 * include/kernix_model.h:560-634). zx: (B*T) x G*u input projections x.W + b of all steps (G = 4, 3, 1); U: u x G*u
 * recurrent weights (row-major as in the file); brec: GRU recurrent bias (G*u); h_prev / h_next: B x u states
 * (h_prev unused when first); c: B x u LSTM cell state; the state at time t goes to out + (b*T + t)*stride when
 * ret_seq, else (when last) to out + b*stride. u <= 12288. */
KERNIX_API int kx_rnn_step(int kind, const float* zx, const float* U, const float* brec, const float* h_prev, float* h_next,
                           float* c, float* out, long stride, int B, int T, int t, int u, int first, int ret_seq, int last,
                           int act, float alpha, void* stream);
/* Merge of a bidirectional RNN's directions in place (kernix_rnn_run :641-646): merge 1 sum, 2 product, 3 average. */
KERNIX_API int kx_rnn_merge(float* y, const float* bw, long n, int merge, void* stream);

/* Dense layer for at most KX_SKINNY_MAX_ROWS rows (weight streaming) on the CUDA cores in fp32:
 * y = act(x . W + bias) with W the k x n row-major fp32 weight as in the file; K is split into kx_skinny_slices(n, k)
 * slices whose partial sums (part: slices x m x n floats) are added in slice order. (Extension; the reference runs
 * every dense layer through one sgemm.) */
#define KX_SKINNY_MAX_ROWS 16
KERNIX_API int kx_skinny_slices(int n, int k);
KERNIX_API int kx_gemm_f32_skinny(const float* x, int ldx, const float* w, const float* bias, float* y, int ldy, int m, int n,
                                  int k, int act, float alpha, float* part, size_t part_floats, void* stream);

#ifdef __cplusplus
}
#endif
#endif
