/*
 * tinybrain_hip.h -- C ABI of TinyBrainHIP, the MI355X (gfx950) backend for
 * TinyBrain's INT8/INT4 weight-only quantized matmul.
 *
 * The ABI is what a Swift `HIPBackend: QuantizedMatMulBackend` binds through
 * a module map (`module CTinyBrainHIP { header "tinybrain_hip.h";
 * link "tinybrain_hip"; export * }`).  Signatures carry plain pointers and
 * sizes only.  All references are to vivekptnk/tinybrain paths.
 *
 * Conventions
 *   - A weight has the reference shape [K, N] = [in_features, out_features]
 *     (QuantizedTensor.shape, Sources/TinyBrainRuntime/QuantizedTensor.swift:73);
 *     x is [M, K] row-major fp32, y is [M, N] row-major fp32.
 *   - Every call returns a tbh_status; on failure tbh_last_error() returns a
 *     message for the calling thread.  A Swift wrapper maps every non-zero
 *     status to `throw`, which keeps the reference's fallback to its CPU path
 *     (QuantizedTensor.swift:630-642).
 */
#ifndef TINYBRAIN_HIP_H
#define TINYBRAIN_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TBH_ABI_VERSION 1

/* ---- status ------------------------------------------------------------ */
typedef int32_t tbh_status;
enum {
    TBH_OK = 0,
    TBH_E_INVALID = 1,      /* bad descriptor, shape mismatch, null pointer */
    TBH_E_UNSUPPORTED = 2,  /* a valid reference input this backend does not take */
    TBH_E_NODEVICE = 3,     /* no usable gfx950 device */
    TBH_E_OOM = 4,          /* device or host allocation failed */
    TBH_E_HIP = 5           /* any other HIP runtime error */
};

/* ---- descriptor codes -------------------------------------------------- */
/* QuantizationPrecision; the values are the TBF precision byte
 * (ModelWeights.swift:395 writes them, :679 reads them). */
enum { TBH_PREC_INT8 = 1, TBH_PREC_INT4 = 2 };

/* QuantizationMode, QuantizedTensor.swift:31-37. */
enum {
    TBH_MODE_SYMMETRIC = 0,        /* INT8, one scale                      */
    TBH_MODE_ASYMMETRIC = 1,       /* INT8, one scale + one zero point     */
    TBH_MODE_PER_CHANNEL = 2,      /* INT8, one scale per output column n  */
    TBH_MODE_INT4 = 3,             /* INT4, one scale per flat group       */
    TBH_MODE_INT4_PER_CHANNEL = 4  /* rejected with TBH_E_UNSUPPORTED: the
                                      reference's dequantize() reads its
                                      scales along dim 0 while its quantizer
                                      writes them along dim 1
                                      (QuantizedTensor.swift:218-238 vs
                                      :563-606), so the caller's CPU
                                      fallback is the only defined result  */
};

/* Order of the flat element array.
 *   KN_FLAT: element (k, n) is flat index k*N + n -- the runtime layout that
 *            Tensor.quantize() writes (QuantizedTensor.swift:379-424,
 *            :502-560) and dequantize() reads (:182-286).
 *   NK_FLAT: element (k, n) is flat index n*K + k -- what
 *            Scripts/convert_model.py:398-459 writes for INT4 (it quantizes
 *            the PyTorch [N, K] tensor flattened and only reverses the
 *            recorded shape, :489-502), i.e. groups run along K.
 * For INT4 the group of flat index i is i / group_size in both layouts. */
enum { TBH_LAYOUT_KN_FLAT = 0, TBH_LAYOUT_NK_FLAT = 1 };

/* struct QuantizedTensor (QuantizedTensor.swift:62-166) as plain data.
 * Counts are checked exactly as QuantizedTensor.init checks them
 * (QuantizedTensor.swift:124-155):
 *   data_bytes    == K*N (INT8) or ceil(K*N/2) (INT4, even flat index in the
 *                    high nibble, QuantizedTensor.swift:201-213)
 *   n_scales      == N (PER_CHANNEL), 1 (SYMMETRIC/ASYMMETRIC),
 *                    ceil(K*N/group_size) (INT4, group_size > 0),
 *                    1 (INT4, group_size == 0: one group of K*N)
 *   n_zero_points == n_scales when zero_points != NULL. */
typedef struct tbh_qtensor_desc {
    int64_t K;
    int64_t N;
    int32_t precision;          /* TBH_PREC_*   */
    int32_t mode;               /* TBH_MODE_*   */
    int32_t layout;             /* TBH_LAYOUT_* */
    int32_t group_size;         /* INT4 only; 0 = single group */
    const int8_t *data;
    int64_t data_bytes;
    const float *scales;
    int64_t n_scales;
    const int8_t *zero_points;  /* nullable (Swift nil) */
    int64_t n_zero_points;
} tbh_qtensor_desc;

/* Which kernel family serves a weight (see tbh_weight_info.path). */
enum {
    TBH_PATH_INT8_ROW = 0,      /* INT8, one scale (and zero point) per row  */
    TBH_PATH_INT4_KGROUP = 1,   /* INT4, scales per (row, K-segment)         */
    TBH_PATH_INT4_NGROUP = 2,   /* INT4 runtime layout, scales per (K, N-block) */
    TBH_PATH_GENERIC = 3        /* any other INT4 grouping: slow, exact decode */
};

typedef struct tbh_weight_info {
    int64_t K;
    int64_t N;
    int32_t precision;
    int32_t mode;
    int32_t layout;
    int32_t group_size;
    int32_t path;               /* TBH_PATH_* */
    int32_t has_zero_points;    /* non-zero zero points were kept */
    int64_t device_bytes;       /* bytes this weight holds in HBM */
    int64_t stream_bytes;       /* bytes one matmul reads from it:
                                   packed weights + scales + zero points */
} tbh_weight_info;

typedef struct tbh_device tbh_device;
typedef struct tbh_weight tbh_weight;

/* ---- library ----------------------------------------------------------- */
int32_t tbh_abi_version(void);
/* Message of the last failure on the calling thread ("" if none). */
const char *tbh_last_error(void);
const char *tbh_status_string(tbh_status status);

/* ---- device ------------------------------------------------------------ */
/* Replaces MetalBackend.init (Sources/TinyBrainMetal/MetalBackend.swift:38-56)
 * and MetalBackend.isAvailable: opens HIP device `ordinal` (must be gfx950)
 * with one internal stream.  TBH_E_NODEVICE when absent. */
tbh_status tbh_device_open(int32_t ordinal, tbh_device **out);
/* Waits for the device's work and frees what the library allocated on it.
 * Destroy the device's weights and decoders first: their destroy calls read
 * the device handle. */
tbh_status tbh_device_close(tbh_device *dev);
/* HIP device ordinal and compute-unit count of an open device. */
tbh_status tbh_device_get_info(const tbh_device *dev, int32_t *ordinal, int32_t *cu_count);

/* Launch-rule overrides of an open device, for measurement and tests.  No
 * reference counterpart (MetalBackend's launch shapes are fixed,
 * MetalBackend.swift:949-956).  Every accepted value keeps results within
 * the matmul tolerance; TBH_E_INVALID for unknown options or values.
 *   TBH_OPT_SGEMV_MIN_ROWS: fewest rows of x (2..9, 9 = never) that go to the
 *     matrix-core small-M GEMV for every weight; 0 restores the per-weight
 *     rule.  The environment variable TBH_SGEMV_MIN_ROWS, read when the
 *     device opens, sets the initial value.
 *   TBH_OPT_NOALLOC_SCRATCH_BYTES: the most scratch bytes
 *     tbh_matmul_device_noalloc may use on this device, 1 .. 16 MiB; 0 (the
 *     default) is the whole 16 MiB array.
 *   TBH_OPT_MFMA_MIN_ROWS: fewest rows of fp32 x that tbh_matmul* send to the
 *     MFMA GEMM (x split exactly into bf16 pieces) for every weight; 0
 *     restores the per-weight rule.
 *   TBH_OPT_HOST_ENTRY: how tbh_matmul moves x and y for up to 8 rows of x:
 *     0 = DMA copies through device staging; 1 = a copy launch brings x from
 *     page-locked staging and the kernels write y into it; 2 (default) = as
 *     1, with one row of x read by the kernels in place.  Initially the
 *     environment variable TBH_HOST_ENTRY when set.
 *   TBH_OPT_HOST_WAIT: how tbh_matmul waits in modes 1 and 2: 1 (default) =
 *     poll a completion word in page-locked memory for up to 200 us, then
 *     block; 0 = block on the stream.  Initially TBH_HOST_WAIT when set. */
enum {
    TBH_OPT_SGEMV_MIN_ROWS = 1,
    TBH_OPT_NOALLOC_SCRATCH_BYTES = 2,
    TBH_OPT_MFMA_MIN_ROWS = 3,
    TBH_OPT_HOST_ENTRY = 4,
    TBH_OPT_HOST_WAIT = 5
};
tbh_status tbh_device_set_option(tbh_device *dev, int32_t option, int64_t value);

/* ---- weights ----------------------------------------------------------- */
/* Replaces the weight upload of MetalBackend.cachedQuantizedBuffers
 * (MetalBackend.swift:1282-1308) and cachedINT4Buffers (:1322-1359): copies
 * the descriptor's arrays and repacks them ONCE into the gfx950 layout; the
 * caller may free its arrays on return.  Thread-safe.  K or N above 2^30
 * returns TBH_E_UNSUPPORTED (the caller's CPU fallback takes it). */
tbh_status tbh_weight_create(tbh_device *dev, const tbh_qtensor_desc *desc,
                             tbh_weight **out);
/* One weight that computes the outputs of n weights reading the same input,
 * side by side: y[M, N_0 + ... + N_{n-1}] = x . [dequantize(W_0) | ... ],
 * repacked once, so that the projections of a layer that read one x (q, k
 * and v; gate and up: ModelRunner.swift:418-452, where each is its own
 * apply(toRow:) call, ModelWeights.swift:47-68) run as one launch.  No
 * single reference counterpart: it is a one-time repack of
 * TransformerLayerWeights' quantized projections.  The parts must share K
 * and precision and be concatenable without re-quantizing: INT8 in the
 * [K][N] layout (per-channel, or a per-tensor scale repeated per column),
 * INT4 in the converter layout (groups along K), or runtime-layout INT4 whose
 * groups tile every part's N; zero points on all parts or none.  Otherwise
 * TBH_E_UNSUPPORTED (or TBH_E_INVALID for inconsistent descriptors).
 * Results are within the matmul tolerance of the parts' products (the
 * kernels chosen for the wider weight may sum in another order). */
tbh_status tbh_weight_create_concat(tbh_device *dev, int32_t n,
                                    const tbh_qtensor_desc *const *parts,
                                    tbh_weight **out);
tbh_status tbh_weight_destroy(tbh_weight *w);
tbh_status tbh_weight_get_info(const tbh_weight *w, tbh_weight_info *info);

/* ---- matmul ------------------------------------------------------------ */
/* Replaces QuantizedMatMulBackend.matmulQuantized
 * (Sources/TinyBrainRuntime/Backend.swift:173-175), implemented by
 * MetalBackend.matmulQuantized / matmulINT4 (MetalBackend.swift:894-1048):
 * y[M,N] = x[M,K] . dequantize(w)[K,N] with fp32 accumulation.
 * Host pointers; synchronous (the reference commits and waits, :959-960).
 * Up to 8 rows of x, the kernels read x from and write y to page-locked
 * host staging, and the calling thread polls a completion word there for up
 * to 200 us before it blocks on the stream; more rows move by DMA.
 * Calls on one device are serialised.  Like the Metal kernels, one call
 * covers any M (MetalBackend.swift:949-956): a few rows run on the GEMV
 * kernels; from a per-weight row count (8..64, TBH_OPT_MFMA_MIN_ROWS) INT8
 * rows, INT4 K-group weights and runtime-layout INT4 whose N-blocks tile 64
 * outputs (16, 32 or a multiple of 64 rows, or one block) run on the bf16
 * MFMA GEMM with every fp32 x row split exactly into three bf16 pieces (for
 * the runtime layout, x times the N-block's per-k scale, one fp32 rounding,
 * then split); past 64 rows x is taken as two f16 pieces, scaled by a power
 * of two per row, holding it to 2^-22 of the row's largest element, on the
 * f16 MFMA.  The GEMV kernels stage a row of
 * x in LDS, so a K past about 13 K (INT8) or 14.5 K (INT4) elements runs on
 * the MFMA GEMM at every M (runtime-layout INT4 of such a K keeps the
 * reference's flat array and runs on the generic kernel); a long K that is
 * not a multiple of 8, or an x that is not 16-byte aligned, returns
 * TBH_E_UNSUPPORTED. */
tbh_status tbh_matmul(tbh_device *dev, const float *x, int64_t M, int64_t K,
                      const tbh_weight *w, float *y);

/* Same product on device pointers, enqueued on `stream` (a hipStream_t of the
 * weight's device; NULL = the null stream).  Returns after the launch.  Host
 * threads may call on one stream: the launches of a call stay together there.
 * Launches that split K (matrix-core GEMV, MFMA GEMM) keep their partial sums,
 * and the MFMA GEMM its 16-bit pieces of fp32 x (4 or 6 bytes per element, up
 * to 128 MiB at a time: longer x is taken in even parts) and their exponents
 * (an int32 per row), in a workspace the library allocates per (device, stream) on first use and
 * keeps, with every buffer it outgrew, until tbh_device_close (a graph
 * captured on the stream may still hold them): a caller that creates many
 * short-lived streams should reuse a few, or call
 * tbh_matmul_device_noalloc.  A graph captured on a stream holds that
 * stream's current workspace, which later eager calls on the same stream
 * reuse: such a graph must not be replayed (on any stream) while eager
 * calls on its capture stream are in flight, or both write the same partial
 * sums. */
tbh_status tbh_matmul_device(const tbh_weight *w, const float *x, int64_t M,
                             int64_t K, float *y, void *stream);

/* No reference counterpart.  tbh_matmul_device for callers that cannot
 * allocate device memory: code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc.  Same product, same kernels, same
 * arguments; the split-K partial sums (matrix-core small-M GEMV, MFMA GEMM)
 * and the GEMM's 16-bit pieces of x go to a fixed 16 MiB scratch array per
 * GPU (held until the process ends) instead of a per-stream workspace, and
 * the call makes no allocation.  The MFMA GEMM past 64 rows, or of a larger
 * weight, takes x and K in parts where the scratch (16 MiB, or
 * TBH_OPT_NOALLOC_SCRATCH_BYTES) does not hold them at once, with the same
 * bits.  A call another launch of which would need more returns TBH_E_INVALID
 * before that launch is enqueued; rows of x that an earlier launch of the
 * same call took on a
 * route without scratch (x runs in pieces of up to 8 rows, and pieces can
 * take different routes) may already have been written, so y is then
 * unspecified (decode shapes need at most a few MiB).  Every call on
 * one GPU shares that GPU's array: calls that overlap on one GPU (different
 * streams, or graphs replayed concurrently) race and must be serialised by
 * the caller. */
tbh_status tbh_matmul_device_noalloc(const tbh_weight *w, const float *x, int64_t M,
                                     int64_t K, float *y, void *stream);

/* Replaces LinearLayerWeights.apply(toRow:)
 * (Sources/TinyBrainRuntime/ModelWeights.swift:47-68): y = x . dequantize(w)
 * as tbh_matmul_device computes it, then y[m][n] += bias[n] (one fp32 add,
 * after the product, as the reference's host loop does).  bias: device
 * pointer to N floats, or NULL for no bias.  Device pointers, enqueued on
 * `stream`. */
tbh_status tbh_linear_device(const tbh_weight *w, const float *x, int64_t M,
                             int64_t K, const float *bias, float *y, void *stream);

/* Prefill: the same product for M >= 64 rows of bf16 activations, on bf16
 * MFMA.  The reference has no bf16 path; it multiplies
 * fp32 activations by dequantize(w) with cblas_sgemm
 * (QuantizedTensor.swift:640-642, Tensor.swift:839-861), which is the
 * product computed here for x = the bf16 values widened to fp32: weight
 * operands are exact integers (INT8: q - zp, the row scale applied after
 * accumulation; INT4 K-groups: 16 (q - zp), each 32-deep MFMA's partial
 * product times its group scale; INT4 runtime layout up to 64 rows: 16 q
 * against x times the N-block's per-k scale, rounded once in fp32 and split
 * exactly into three bf16 pieces), accumulation is fp32.  INT4 runtime
 * layout past 64 rows runs on f16 MFMA: the dequantized weight fl(q * s),
 * scaled by a power of two per N-block, as two f16 pieces holding it to
 * 2^-21 of itself, against x scaled by a power of two per row (exact), a pass
 * that writes x so, 2 bytes per element, to the stream's workspace.  x is [M, K] row-major bf16 bits
 * (16-byte aligned, K % 8 == 0), y is [M, N] fp32, both device pointers;
 * enqueued on `stream`.  TBH_E_UNSUPPORTED for weights outside the INT8
 * row / INT4 K-group / INT4 runtime-layout paths (tbh_weight_info.path), for
 * runtime-layout N-blocks that do not tile 64 outputs, or for the MFMA tile
 * layout. */
tbh_status tbh_matmul_bf16_device(const tbh_weight *w, const uint16_t *x, int64_t M,
                                  int64_t K, float *y, void *stream);

/* ---- decode step (LLaMA-style models, one sequence) -------------------- */
/* Replaces ModelRunner.step (Sources/TinyBrainRuntime/ModelRunner.swift:168-208)
 * for the pre-norm LLaMA architecture (applyLayer :418-459, attention
 * :496-592): RMSNorm, Q/K/V, RoPE, grouped-query attention over a KV cache,
 * output projection and residual, RMSNorm, SwiGLU FFN and residual, final
 * RMSNorm and the LM head, every projection on the quantized GEMV.  Gemma /
 * Phi variants, biases and X-Ray observers are not covered.  The position is
 * kept on the device and advanced by each step, so a step captured in a HIP
 * graph replays as the next one. */
typedef struct tbh_decoder tbh_decoder;
typedef struct tbh_decoder_config {
    int32_t num_layers;
    int32_t hidden;          /* ModelConfig.hiddenDim */
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t intermediate;    /* ModelConfig.intermediateDim */
    int32_t vocab;
    int32_t max_seq;         /* KV cache length, <= 16384 */
    float rms_eps;           /* 1e-5 (Tensor.swift:1512) */
    float rope_base;         /* 10000 (ModelRunner.swift:478) */
} tbh_decoder_config;

/* embeddings: [vocab][hidden] fp32 (ModelWeights.tokenEmbeddings);
 * final_norm: [hidden]; lm_head: [hidden, vocab] (ModelWeights.output).
 * Host pointers, copied. */
tbh_status tbh_decoder_create(tbh_device *dev, const tbh_decoder_config *cfg,
                              const float *embeddings, const float *final_norm,
                              const tbh_qtensor_desc *lm_head, tbh_decoder **out);
/* One TransformerLayerWeights (ModelWeights.swift): norms [hidden] and the
 * seven projections as [K, N] quantized tensors (q [hidden, hidden], k and v
 * [hidden, kv_dim], o [hidden, hidden], gate and up [hidden, intermediate],
 * down [intermediate, hidden]).  Q|K|V and gate|up are concatenated along N
 * into one repacked weight each.  Needs weights without zero points: INT8
 * in the runtime layout, INT4 in the converter layout (groups along K) or
 * INT4 in the runtime layout (Tensor.quantize(.int4), groups along N) whose
 * groups tile every projection's N. */
tbh_status tbh_decoder_set_layer(tbh_decoder *d, int32_t layer, const float *input_norm,
                                 const float *post_attention_norm,
                                 const tbh_qtensor_desc *q, const tbh_qtensor_desc *k,
                                 const tbh_qtensor_desc *v, const tbh_qtensor_desc *o,
                                 const tbh_qtensor_desc *gate, const tbh_qtensor_desc *up,
                                 const tbh_qtensor_desc *down);
tbh_status tbh_decoder_destroy(tbh_decoder *d);
/* ModelRunner.reset (:213-216) is set_position(d, 0). */
tbh_status tbh_decoder_set_position(tbh_decoder *d, int32_t position);
tbh_status tbh_decoder_get_position(const tbh_decoder *d, int32_t *position);
/* Enqueue one step for `token` on `stream`; logits: device [vocab] (NULL:
 * internal buffer). */
tbh_status tbh_decoder_step_device(tbh_decoder *d, int32_t token, float *logits, void *stream);
/* Synchronous step; logits: host [vocab]. */
tbh_status tbh_decoder_step(tbh_decoder *d, int32_t token, float *logits);

/* ---- TBF v1 model files ------------------------------------------------ */
/* Reader of the .tbf files ModelWeights.save writes and ModelWeights.load
 * reads (Sources/TinyBrainRuntime/ModelWeights.swift:376-488, :496-798), and
 * Scripts/convert_model.py:462-706 writes.  The file is memory-mapped and
 * every field bounds-checked (malformed: TBH_E_INVALID).  Descriptors and
 * fp32 pointers point into the mapping and stay valid until tbh_tbf_close. */
typedef struct tbh_tbf tbh_tbf;
typedef struct tbh_tbf_config {    /* ModelConfig (ModelRunner.swift:26-120) */
    int32_t num_layers;
    int32_t hidden;
    int32_t num_heads;
    int32_t num_kv_heads;          /* default num_heads */
    int32_t vocab;
    int32_t max_seq;
    int32_t intermediate;          /* default 4 * hidden */
    float partial_rotary_factor;   /* default 1.0 */
    char architecture[16];         /* default "llama" */
} tbh_tbf_config;
typedef struct tbh_tbf_tensor_info {
    const char *name;              /* owned by the file handle */
    int32_t ndim;
    int32_t quantized;             /* has a quantization metadata entry */
    int64_t dims[4];
    int64_t offset;                /* absolute file offset of the blob */
    int64_t bytes;
} tbh_tbf_tensor_info;

tbh_status tbh_tbf_open(const char *path, tbh_tbf **out);
tbh_status tbh_tbf_close(tbh_tbf *f);
tbh_status tbh_tbf_get_config(const tbh_tbf *f, tbh_tbf_config *cfg);
int32_t tbh_tbf_tensor_count(const tbh_tbf *f);
tbh_status tbh_tbf_tensor(const tbh_tbf *f, int32_t index, tbh_tbf_tensor_info *t);
tbh_status tbh_tbf_find(const tbh_tbf *f, const char *name, int32_t *index);
/* The quantized tensor as ModelWeights.load builds it (:676-685): precision
 * 2 is INT4 (layout NK_FLAT when the converter wrote it, mode byte 3;
 * KN_FLAT when ModelWeights.save did, mode byte 2); INT8 mode 2 is
 * per-channel, other INT8 modes symmetric. */
tbh_status tbh_tbf_qtensor(const tbh_tbf *f, int32_t index, tbh_qtensor_desc *desc);
tbh_status tbh_tbf_floats(const tbh_tbf *f, int32_t index, const float **data, int64_t *count);
/* A decoder for a LLaMA-architecture file (ModelWeights.load followed by
 * ModelRunner): every quantized projection repacked once; max_seq 0 = the
 * file's maxSeqLen.  TBH_E_UNSUPPORTED for other architectures, biases or an
 * ungated FFN. */
tbh_status tbh_tbf_load_decoder(tbh_device *dev, const tbh_tbf *f, int32_t max_seq,
                                tbh_decoder **out);

/* ---- dequantize (verification) ----------------------------------------- */
/* Replaces QuantizedTensor.dequantize() (QuantizedTensor.swift:182-286) for
 * the uploaded weight: writes the [K, N] row-major fp32 matrix that the
 * matmul multiplies by, bit-identical to (float)(q - zp) * scale.  For
 * KN_FLAT weights this is exactly the reference's dequantize() output; for
 * NK_FLAT INT4 it is that output read in the converter's [N, K] order and
 * transposed.  Host pointer, synchronous. */
tbh_status tbh_dequantize(tbh_device *dev, const tbh_weight *w, float *out);
tbh_status tbh_dequantize_device(const tbh_weight *w, float *out, void *stream);

/* ---- the other backend protocols (Backend.swift:177-228) --------------- */
/* Each op has a host-pointer call (synchronous, serialised per device, like
 * tbh_matmul) and a _device call (device pointers, enqueued on a hipStream_t
 * and returning after the launch).  Sizes of 0 are no-ops.  Results are fp32
 * computed in fp32. */

/* SoftmaxBackend.softmax (Backend.swift:180-186; MetalBackend.swift:1073-1134,
 * Shaders/Softmax.metal): each of `rows` rows of `cols` elements becomes
 * exp(x - max) / (sum + 1e-7), the epsilon of Tensor.softmaxCPU
 * (Tensor.swift:1271-1330). */
tbh_status tbh_softmax(tbh_device *dev, const float *x, int64_t rows, int64_t cols, float *y);
tbh_status tbh_softmax_device(tbh_device *dev, const float *x, int64_t rows, int64_t cols, float *y,
                              void *stream);

/* RMSNormBackend.rmsnorm (Backend.swift:188-199; MetalBackend.swift:1146-1207):
 * per row of `hidden` elements, y = x * (1 / sqrt(sum(x^2) / hidden + eps)) *
 * weight, as Tensor.rmsNormCPU (Tensor.swift:1538-1556). */
tbh_status tbh_rmsnorm(tbh_device *dev, const float *x, int64_t rows, int64_t hidden, const float *weight,
                       float eps, float *y);
tbh_status tbh_rmsnorm_device(tbh_device *dev, const float *x, int64_t rows, int64_t hidden,
                              const float *weight, float eps, float *y, void *stream);

/* ActivationBackend (Backend.swift:222-228): silu y = x / (1 + exp(-x))
 * (Tensor.swift:1135-1141); gelu, tanh form, y = 0.5 x (1 + tanh(sqrt(2/pi)
 * (x + 0.044715 x^3))) (Tensor.swift:1107-1121). */
tbh_status tbh_silu(tbh_device *dev, const float *x, int64_t n, float *y);
tbh_status tbh_silu_device(tbh_device *dev, const float *x, int64_t n, float *y, void *stream);
tbh_status tbh_gelu(tbh_device *dev, const float *x, int64_t n, float *y);
tbh_status tbh_gelu_device(tbh_device *dev, const float *x, int64_t n, float *y, void *stream);

/* AttentionBackend.attention (Backend.swift:201-220; MetalBackend.swift:1381-1525,
 * Shaders/FlashAttention.metal).  q [batch][seq_len][num_heads * head_dim],
 * k and v [batch][kv_len][num_kv_heads * head_dim], optional additive mask
 * [kv_len] shared by every query (0 attends, -inf ignores), out shaped like
 * q.  Query head h reads key/value head h / (num_heads / num_kv_heads);
 * scores are q.k / sqrt(head_dim) + mask; out = sum(p v) / (sum(p) + 1e-7)
 * with p = exp(score - max) over all kv_len positions.  A row whose
 * positions are all masked gives NaN, as the reference's CPU attention does;
 * kv_len 0 gives zeros. 
 * num_heads must be a multiple of num_kv_heads; head_dim <= 256. */
typedef struct tbh_attention_shape {
    int64_t batch;
    int64_t seq_len;
    int64_t kv_len;
    int32_t head_dim;
    int32_t num_heads;
    int32_t num_kv_heads;
} tbh_attention_shape;

tbh_status tbh_attention(tbh_device *dev, const tbh_attention_shape *shape, const float *q, const float *k,
                         const float *v, const float *mask, float *out);
tbh_status tbh_attention_device(tbh_device *dev, const tbh_attention_shape *shape, const float *q,
                                const float *k, const float *v, const float *mask, float *out, void *stream);

/* ---- serving many requests from one paged cache ------------------------ */
/* The decode step above keeps the cache of one sequence.  These calls serve a
 * batch: requests of any lengths share one key/value cache cut into blocks of
 * block_size tokens (the reference's KVCache is paged too, 16 tokens a page,
 * but holds one sequence: KVCache.swift:61-120).  One step of a batch is
 *   tbh_paged_plan_device       lengths -> blocks, slots, positions (once)
 *   tbh_paged_append_device     a layer's new keys and values -> the cache
 *   tbh_paged_attention_device  the layer's attention over the cache
 *   tbh_sample_device           logits -> tokens
 * All of them take device pointers, are enqueued on `stream` and return after
 * the launch; lengths, tables and slots are read on the device, so a captured
 * step replays with new ones.  Host threads may call on one stream: the
 * launches of a call stay together there.  Device-side values out of range are never
 * followed: a block id outside the cache holds nothing, a slot outside it is
 * not written, lengths are clamped to what the table and the rows can hold.
 *
 * The cache of a layer is two arrays (keys, values), each
 * [num_blocks][num_kv_heads][block_size][head_dim] of `type`, 16-byte aligned.
 * Request b is row b of block_table [max_requests][max_blocks]; its position p
 * lies in block block_table[b][p / block_size] at row p % block_size, and the
 * slot of that place is block * block_size + p % block_size. */
enum { TBH_F32 = 0, TBH_BF16 = 1 };   /* element types of the cache, of rows and of activations */

typedef struct tbh_paged_layout {
    int32_t num_blocks;      /* blocks in each array; num_blocks * block_size < 2^31 */
    int32_t block_size;      /* tokens per block: a power of two, 1 .. 1024 */
    int32_t num_kv_heads;
    int32_t head_dim;        /* 1 .. 256 */
    int32_t type;            /* TBH_F32 or TBH_BF16 */
    int32_t max_requests;    /* rows of the block table, at most 2^30 */
    int32_t max_blocks;      /* entries per row; max_blocks * block_size <= 2^30 */
} tbh_paged_layout;

/* Plans a step.  new_lens[max_requests]: tokens each request adds (0: idle
 * this step; negative: the request is released).  context_lens: tokens each
 * holds so far, in the first ceil(context / block_size) blocks of its row.
 * free_blocks[num_blocks] is a stack of free block ids, free_count[1] its
 * height.  In order:
 *   - released rows push their blocks (row by row, in table order);
 *   - row b with n = new_lens[b] > 0 needs ceil((context + n) / block_size) -
 *     ceil(context / block_size) blocks and is granted its tokens if context +
 *     n fits the table row, query_start[b] + n fits max_tokens, and the needs
 *     of rows 0 .. b (of those that fit both) do not exceed the stack, or it
 *     needs none: no row overtakes one that waits for blocks, and rows behind
 *     one whose tokens pass max_tokens wait with it;
 *   - granted rows pop their blocks off the stack (row by row) into the table.
 * Outputs: query_start[max_requests + 1], running sums of max(new_lens, 0);
 * granted[max_requests], n or 0; context_out, free_count_out: the lengths and
 * the height after the step; slots[max_tokens], positions[max_tokens] of token
 * query_start[b] + i, position context[b] + i, and -1 for rows not granted and
 * for entries behind the last token.
 * context_out and free_count_out may be context_lens and free_count; else a
 * plan can be dropped: entries of the table and of the stack that the old
 * lengths and height refer to are not changed.  Only the block_size, num_blocks,
 * max_requests and max_blocks of the layout are read. */
tbh_status tbh_paged_plan_device(tbh_device *dev, const tbh_paged_layout *layout, const int32_t *new_lens,
                                 const int32_t *context_lens, int32_t *block_table, int32_t *free_blocks,
                                 const int32_t *free_count, int64_t max_tokens, int32_t *query_start,
                                 int32_t *granted, int32_t *context_out, int32_t *free_count_out,
                                 int32_t *slots, int32_t *positions, void *stream);

/* Rows of a projection on their way to the attention and the cache. */
typedef struct tbh_paged_rows {
    int64_t tokens;
    int32_t x_type;          /* of q, k and v */
    int32_t num_heads;       /* of q */
    const void *q;           /* [tokens][num_heads * head_dim], or NULL */
    const void *k;           /* [tokens][num_kv_heads * head_dim] */
    const void *v;           /* as k */
    int64_t q_stride;        /* elements from one row to the next */
    int64_t k_stride;
    int64_t v_stride;
    void *q_out;             /* [tokens][num_heads * head_dim]; may be q itself (same type and stride), */
                             /* else it overlaps none of q, k and v */
    int64_t q_out_stride;
    int32_t q_out_type;
    float rope_base;         /* 0: no rotation */
    const int32_t *slots;    /* [tokens]; distinct, or negative: the row is not stored */
    const int32_t *positions;/* [tokens]; read with rope_base > 0, negative as 0 */
} tbh_paged_rows;

/* Stores the rows' keys and values at their slots, rounded once to the
 * cache's type, and, with rope_base > 0, rotates keys and queries first:
 * interleaved pairs (2i, 2i + 1) by the angle position * rope_base^(-2i /
 * head_dim), as ModelRunner.applyRoPE (ModelRunner.swift:470-494).  The angle
 * is that of real arithmetic (the reference, and the decode step here, round
 * it to fp32, which at position 10^5 is off by up to 4e-3).  q NULL: no
 * queries.  An odd head_dim is not rotated (TBH_E_INVALID). */
tbh_status tbh_paged_append_device(tbh_device *dev, const tbh_paged_layout *layout, const tbh_paged_rows *rows,
                                   void *k_cache, void *v_cache, void *stream);

/* A batch of queries over the cache. */
typedef struct tbh_paged_queries {
    int64_t tokens;              /* rows of q and out */
    int32_t type;                /* of q and out */
    int32_t num_heads;
    const void *q;               /* [tokens][num_heads * head_dim] */
    void *out;                   /* as q, not overlapping it */
    int64_t q_stride;
    int64_t out_stride;
    const int32_t *query_start;  /* [max_requests + 1], not negative, not descending */
    const int32_t *context_lens; /* [max_requests], with the step's own tokens */
    float scale;                 /* of the scores; 0: 1 / sqrt(head_dim) */
    int32_t max_query_len;       /* at least the longest query_start[b + 1] - query_start[b], */
    int32_t max_context_len;     /* and the longest context: they choose launch shapes only; 0: unknown */
} tbh_paged_queries;

/* Attention of each request's newest tokens over its cache: row i of request
 * b's n rows has position context_lens[b] - n + i and attends to every
 * position up to its own, out = sum softmax(scale q . k) v per head, query
 * head h reading key/value head h / (num_heads / num_kv_heads).  Prompt
 * chunks and single tokens mix in one call.  A row with nothing to attend to
 * (negative position, no block) gives zeros; rows before query_start's first
 * entry or behind its last are left as they are.  Whatever lies in the cache behind a request's
 * length is not used (it may be NaN).  Scores, softmax and sums are fp32; fp32
 * q keeps fp32's precision over a bf16 cache as well, bf16 q over a bf16 cache
 * has its probabilities rounded to bf16 for the second product.
 * num_heads must be a multiple of num_kv_heads.  Calls that split a long
 * context over blocks keep partial results in the workspace of (device,
 * stream), as tbh_matmul_device does, with its rule for captured graphs: at
 * most 256 MiB, for which the bounds on the lengths count, not the lengths
 * themselves (contexts are cut into fewer parts where more would be needed).
 * Without a workspace (none can be had, or it would have to grow under
 * capture) contexts are not cut. */
tbh_status tbh_paged_attention_device(tbh_device *dev, const tbh_paged_layout *layout,
                                      const tbh_paged_queries *queries, const void *k_cache, const void *v_cache,
                                      const int32_t *block_table, void *stream);

/* ---- products with block-scaled FP8 weights ------------------------------ */
/* A third stored format beside INT8 and INT4 (no reference counterpart: its
 * weights are INT8 or INT4): e4m3 bytes (1 sign, 4 exponent, 3 mantissa bits,
 * largest value 448, no infinities; 0x7F and 0xFF are NaN) with one fp32 scale
 * for each block of 128 outputs by 128 inputs.  Element (k, n) of the [K, N]
 * weight is data[n * K + k] * scales[(n / 128) * ceil(K / 128) + k / 128].
 * data and scales may be host or device pointers; device data has to be there
 * before the call.  Copied and repacked once. */
typedef struct tbh_fp8_desc {
    int64_t K;                  /* up to 2^20 */
    int64_t N;                  /* up to 2^24 */
    const uint8_t *data;        /* [N][K] */
    const float *scales;        /* [ceil(N / 128)][ceil(K / 128)] */
} tbh_fp8_desc;
typedef struct tbh_fp8_weight tbh_fp8_weight;
tbh_status tbh_fp8_weight_create(tbh_device *dev, const tbh_fp8_desc *desc, tbh_fp8_weight **out);
/* Destroy before the device is closed, as weights are. */
tbh_status tbh_fp8_weight_destroy(tbh_fp8_weight *w);

/* y[M, N] = x[M, K] . W[K, N] in 8-bit floating point: x (TBH_F32 or TBH_BF16,
 * rows x_stride elements apart) is quantized to e4m3 as well, with a scale for
 * each row and block b of 128 inputs: s = the least power of two (at least
 * 2^-126) with |x| <= 448 s over the block's finite elements, q = x / s rounded
 * once, ties to even; an infinity or NaN becomes NaN.
 *   y[m][n] = sum over b of s[m][b] * scale[n / 128][b] * (q . w of block b)
 * summed in fp32, rounded once to y_type.  For TBH_BF16 q . w comes from the FP8
 * matrix instruction, which cuts its sums (about 2^-15 of their size, at most 2^-10
 * of a block's largest product; rounding to bf16 then does 2^-9); TBH_F32 results
 * have fp32 sums, on the bf16 instruction, to which q and w are widened exactly.
 * (Products of two scales outside fp32's normal range lose precision or overflow.)
 * y does not overlap x.
 * Past 16 rows x is quantized into `workspace` (256-byte aligned,
 * tbh_fp8_matmul_workspace bytes for M rows), or, if that is NULL, into the
 * workspace of (device, stream), with tbh_matmul_device's rule for captured
 * graphs; where none can be had (a capture before any eager call on its
 * stream) the rows run 16 at a time without it. */
tbh_status tbh_fp8_matmul_workspace(const tbh_fp8_weight *w, int64_t M, int64_t *bytes);
tbh_status tbh_fp8_matmul_device(const tbh_fp8_weight *w, const void *x, int32_t x_type, int64_t M, int64_t K,
                                 int64_t x_stride, void *y, int32_t y_type, int64_t y_stride, void *workspace,
                                 int64_t workspace_bytes, void *stream);

/* ---- mixture-of-experts layer ---------------------------------------------- */
/* The feed-forward layer of a mixture-of-experts model on block-scaled FP8
 * weights, beside the dense one of the decode step (no reference counterpart:
 * its FFN is dense, ModelRunner.swift:445-457).  For a token's row x:
 *   z = x . router^T in 64-bit sums; its experts are the top_k largest z (of
 *   equal ones the lowest), with weights p_e = exp(z_e) / sum of exp(z) over
 *   all experts, or over the chosen ones (normalize)
 *   y = sum over its experts of p_e (silu(x . G_e) * (x . U_e)) . D_e
 * Activations are not quantized: bf16 rows are taken as they are (h is held to
 * 2^-16 of itself, y is rounded to bf16 once, from fp32), fp32 rows keep fp32's
 * precision throughout.
 * Made for few tokens, where reading the chosen experts is what takes time: an
 * expert's weights are read from memory once for up to 64 tokens, more run 64 at a
 * time.
 * A row that holds an infinity or NaN gets NaN; which experts it is given then
 * means nothing.  Other rows are not touched by it.  An h past the largest fp32
 * number is an infinity and weighs like one. */
typedef struct tbh_moe_desc {
    int32_t hidden;             /* H, up to 2^17 */
    int32_t intermediate;       /* I, up to 2^17 */
    int32_t experts;            /* E, up to 512 */
    int32_t reserved;           /* 0 */
    const float *router;        /* [E][H] */
    const uint8_t *gate;        /* [E][I][H] e4m3, each expert as a tbh_fp8_desc's data */
    const uint8_t *up;          /* [E][I][H] */
    const uint8_t *down;        /* [E][H][I] */
    const float *gate_scales;   /* [E][ceil(I / 128)][ceil(H / 128)] */
    const float *up_scales;
    const float *down_scales;   /* [E][ceil(H / 128)][ceil(I / 128)] */
} tbh_moe_desc;
typedef struct tbh_moe tbh_moe;
/* Host or device pointers, copied and repacked once (as tbh_fp8_weight_create). */
tbh_status tbh_moe_create(tbh_device *dev, const tbh_moe_desc *desc, tbh_moe **out);
tbh_status tbh_moe_destroy(tbh_moe *m);
/* x and y: [tokens][H] of x_type, rows x_stride and y_stride elements apart; y
 * does not overlap x.  experts, weights [tokens][top_k] (each may be NULL):
 * what the router chose, largest first; they overlap neither x, y nor each
 * other.  top_k up to 32.  workspace:
 * 256-byte aligned, tbh_moe_workspace bytes, of which the first
 * TBH_WORKSPACE_COUNTERS are zero (calls leave them so), or NULL for the one of
 * (device, stream), with tbh_matmul_device's rule for captured graphs; a capture
 * before any eager call on its stream finds none (TBH_E_OOM). */
enum { TBH_WORKSPACE_COUNTERS = 32768 };
tbh_status tbh_moe_workspace(const tbh_moe *m, int32_t x_type, int64_t tokens, int32_t top_k, int64_t *bytes);
tbh_status tbh_moe_device(const tbh_moe *m, const void *x, int32_t x_type, int64_t tokens, int64_t x_stride,
                          int32_t top_k, int32_t normalize, void *y, int64_t y_stride, int32_t *experts,
                          float *weights, void *workspace, int64_t workspace_bytes, void *stream);

/* ---- sampling ---------------------------------------------------------- */
/* Sampler (Sampler.swift) with the random numbers given by the caller: one
 * token per row of `logits` [rows][ld] (ld >= vocab).  With w_i =
 * exp((logit_i - max) / temperature):
 *   top_k  > 0 keeps the top_k largest logits (equal ones: lowest index first);
 *   top_p  < 1 keeps of those, largest first, the shortest prefix whose w sum
 *          to at least top_p of their sum (at least one);
 *   min_p  > 0 keeps of those the ones with w_i >= min_p;
 * tokens[r] is the first kept j, in index order, with sum of w over kept i <= j
 * above u[r] times the sum of all kept; probs[r] (if not NULL) is its share of
 * that sum.  temperature <= 0 (or NaN) takes the largest logit, the first of
 * equal ones, with probability 1.  NaN and -inf are never taken (+inf shares
 * all of the weight); a row of nothing else gives token -1, probability 0.
 * u is clamped to [0, 1).  temperature, top_k, top_p, min_p: [rows] each, or
 * NULL for 1, 0, 1, 0 everywhere; NaN top_p or min_p filter nothing, and the
 * largest logit always stays.  Weights are summed as whole multiples of 2^-43 of
 * the largest (64-bit integers), so results do not depend on the order of sums;
 * what weighs less than half of that is never taken.
 * vocab up to 2^20 (TBH_E_UNSUPPORTED above). */
tbh_status tbh_sample(tbh_device *dev, const float *logits, int64_t rows, int64_t vocab, const float *temperature,
                      const int32_t *top_k, const float *top_p, const float *min_p, const float *u,
                      int32_t *tokens, float *probs);
tbh_status tbh_sample_device(tbh_device *dev, const float *logits, int64_t ld, int64_t rows, int64_t vocab,
                             const float *temperature, const int32_t *top_k, const float *top_p,
                             const float *min_p, const float *u, int32_t *tokens, float *probs, void *stream);

/* ---- beam search -------------------------------------------------------------- */
/* Beside sampling, the other way to go on (no reference counterpart: its Sampler
 * draws one token).  Request r has the rows r * beams .. r * beams + beams - 1
 * of logits [requests * beams][ld] (ld >= vocab), scores (the sums of log
 * probabilities so far) and done (nonzero: the row has ended; NULL: none).  Its
 * candidates are, of each row b,
 *   not done: every token j, with scores[b] + logit_j - log(sum of exp(logit))
 *   done:     the token eos, with scores[b]
 * and the k best of them, best first, are its tokens, parents (rows, as
 * counted over the whole call) and scores_out, [requests][k] each; equal ones:
 * the lowest row, then the lowest token.  Candidates are computed and compared in
 * 64 bits (exp to some 1e-12), the same for equal rows.
 * done_out (or NULL) [requests][k]: 1 for the token eos and children of a done
 * row.  NaN and -inf logits are never taken and weigh nothing (+inf ones share
 * all of the weight); a row whose score is not finite has no candidates.  Where
 * there are fewer than k: token and parent -1, score -inf, not done.
 * With scores, done and parents of one call as the next one's, k = beams.
 * The outputs overlap no input and no other output, but for scores_out, which
 * may be scores where k = beams.  beams and k up to 64, vocab and rows up to
 * 2^20 (TBH_E_UNSUPPORTED).  workspace: as tbh_moe_device's, of
 * tbh_beam_select_workspace bytes. */
tbh_status tbh_beam_select_workspace(tbh_device *dev, int64_t requests, int32_t beams, int64_t vocab, int32_t k,
                                     int64_t *bytes);
tbh_status tbh_beam_select_device(tbh_device *dev, const float *logits, int64_t ld, int64_t requests, int32_t beams,
                                  int64_t vocab, const float *scores, const int32_t *done, int32_t eos, int32_t k,
                                  int32_t *tokens, int32_t *parents, float *scores_out, int32_t *done_out,
                                  void *workspace, int64_t workspace_bytes, void *stream);

/* The paged cache after a selection: row i of the block table goes on where row
 * parents[i] stood.  Rows come in groups of `beams` (up to 64), parents lie in
 * their own group; -1: nobody's child.  In each group
 *   - a parent's table row goes to itself if it is its own child, else to its
 *     first child;
 *   - the other rows get the table rows that no parent holds, in order, and the
 *     contents of their parent's positions shared_lens[group] (rounded down to
 *     whole blocks; NULL: 0) .. context are copied into those blocks, in every
 *     layer's arrays.  Positions before shared_lens are taken to be the same in
 *     the whole group: a prompt's, whose whole blocks rows may share; of the
 *     others each stands in one place of the table only.
 * So blocks stay with the group and nothing is allocated.  The rows of a group
 * hold equally many tokens (context_lens); a group whose rows do not, or with a
 * parent outside it, is left as it is.  reordered[groups] (or NULL): 1, or 0 for
 * such a group.  table_out [max_requests][max_blocks] is block_table itself or
 * does not overlap it.  k_caches and v_caches: host arrays of `layers` device
 * pointers.  Places behind a context are not touched.  Block ids outside the
 * cache are not followed. */
tbh_status tbh_paged_reorder_device(tbh_device *dev, const tbh_paged_layout *layout, int32_t beams,
                                    const int32_t *parents, const int32_t *context_lens, const int32_t *shared_lens,
                                    const int32_t *block_table, int32_t *table_out, int32_t layers,
                                    void *const *k_caches, void *const *v_caches, int32_t *reordered, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* TINYBRAIN_HIP_H */
