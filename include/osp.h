/* libosp_hip -- C ABI of the MI355X-native OptiSpeech hot path (generated by tools/gen_header.py; do not edit).
 *
 * Conventions
 *   - every entry point is extern "C", returns int (0 = OSP_OK, < 0 = error; text via osp_last_error()),
 *     never throws, never allocates, never synchronises: work is enqueued on the caller's hipStream_t;
 *     `*_workspace_*` queries return sizes and take no stream
 *   - pointers are DEVICE pointers; activations are channels-last (B, T, C) contiguous f32; utterance lengths are
 *     int64 device arrays; sizes are int64_t, real scalars float
 *   - parameter gradients are ACCUMULATED (+=, f32 atomics) into the caller's gradient arena
 *   - "replaces:" names the reference interface (file:line in mush42/optispeech @ 2024-12-20) each call stands in for
 */
#ifndef OSP_H
#define OSP_H
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif
typedef struct ihipStream_t* hipStream_t;

#define OSP_OK 0
#define OSP_ERR_ARG (-1)
#define OSP_ERR_HIP (-2)
#define OSP_ERR_UNSUPPORTED (-3)

/* epilogues of osp_conv_gemm_* */
enum { OSP_EPI_NONE = 0, OSP_EPI_RELU = 1, OSP_EPI_GELU = 2, OSP_EPI_SCALE_RES_MASK = 3, OSP_EPI_GELU_BWD = 4,
       OSP_EPI_RELU_BWD = 5, OSP_EPI_AXMY = 6, OSP_EPI_MASK = 7, OSP_EPI_LRELU = 8, OSP_EPI_LRELU_BWD = 9 };

/* ---- a16_conv.hip ---- */
/* replaces: CausalConv1d / nn.Conv1d(dilation=d): vocoder/streaming_hifigan/modules/conv_layer.py:18-60,118-159 (callers residual_block.py:44-70) */
int osp_conv1d_dilated_fwd(const void* x, int64_t x_bf16, const void* w, int64_t w_bf16, const float* bias, void* y, int64_t y_bf16, int64_t B, int64_t T, int64_t Cin, int64_t Cout, int64_t k, int64_t dil, int64_t pad_left, int64_t accumulate, hipStream_t stream);

/* replaces: autograd of the same (input, weight and bias gradients) */
int osp_conv1d_dilated_bwd(const void* dy, int64_t dy_bf16, const void* x, int64_t x_bf16, const void* w, int64_t w_bf16, void* dx, int64_t dx_bf16, float* dw, float* db, int64_t B, int64_t T, int64_t Cin, int64_t Cout, int64_t k, int64_t dil, int64_t pad_left, int64_t accumulate_dx, hipStream_t stream);

/* replaces: CausalConvTranspose1d / nn.ConvTranspose1d(stride s): vocoder/streaming_hifigan/modules/conv_layer.py:63-115,162-200 */
int osp_conv_transpose1d_fwd(const void* x, int64_t x_bf16, const void* wn, int64_t w_bf16, const float* bias, void* y, int64_t y_bf16, int64_t B, int64_t T, int64_t Cin, int64_t Cout, int64_t k, int64_t s, int64_t accumulate, hipStream_t stream);

/* replaces: autograd of the same (input and weight gradients) */
int osp_conv_transpose1d_bwd(const void* dy, int64_t dy_bf16, const void* x, int64_t x_bf16, const void* wt, int64_t w_bf16, void* dx, int64_t dx_bf16, float* dwt, int64_t B, int64_t T, int64_t Cin, int64_t Cout, int64_t k, int64_t s, int64_t accumulate_dx, hipStream_t stream);

/* ---- align.hip ---- */
/* replaces: scipy.special gammaln inside scipy.stats.betabinom.logpmf (alignments.py:114) */
int osp_lgamma_table(double* out, int64_t n, hipStream_t stream);

/* replaces: AlignmentModule._generate_prior generator/alignments.py:85-123 */
int osp_betabinom_prior(const double* lg, int64_t lg_len, const int64_t* x_len, const int64_t* y_len, float* out, int64_t B, int64_t Tm, int64_t Nm, hipStream_t stream);

/* replaces: AlignmentModule.forward generator/alignments.py:66-72 */
int osp_pairwise_score(const float* f, const float* e, const int64_t* x_len, float* score, int64_t B, int64_t Tm, int64_t Nm, int64_t C, hipStream_t stream);

/* replaces: AlignmentModule.forward generator/alignments.py:74-81 */
int osp_logsoftmax_prior_fwd(const float* score, const float* prior, float* lp, float* lse, int64_t rows, int64_t Nm, hipStream_t stream);

/* replaces: autograd of generator/alignments.py:66-81 */
int osp_logsoftmax_prior_bwd(const float* dlp, const float* score, const float* lse, const int64_t* x_len, const int64_t* y_len, float* w, float* wrow, int64_t B, int64_t Tm, int64_t Nm, hipStream_t stream);

/* replaces: workspace query for osp_mas */
int64_t osp_mas_workspace_bytes(int64_t B, int64_t Tm, int64_t Nm);

/* replaces: _monotonic_alignment_search + viterbi_decode generator/alignments.py:177-239 (numba JIT + np.bincount) */
int osp_mas(const float* lp, const int64_t* x_len, const int64_t* y_len, int* path, float* durations, float* bin_sum, void* workspace, int64_t B, int64_t Tm, int64_t Nm, hipStream_t stream);

/* replaces: autograd of `bin_loss - cur_log_p_attn[t_idx, viterbi].mean()` generator/alignments.py:236-238 */
int osp_bin_loss_bwd(const int* path, const int64_t* y_len, const float* gscale, float* dlp, int64_t B, int64_t Tm, int64_t Nm, hipStream_t stream);

/* replaces: _average_by_duration / average_by_duration generator/alignments.py:242-280; cumsum at :167 */
int osp_duration_stats(const float* ds, const float* xs0, const float* xs1, const int64_t* x_len, const int64_t* y_len, float* avg0, float* avg1, float* centre, int64_t B, int64_t Tm, int64_t Nm, hipStream_t stream);

/* replaces: GaussianUpsampling.forward generator/alignments.py:163-172 */
int osp_gaussian_weights(const float* centre, const int64_t* x_len, const int64_t* y_len, float delta, float* P, int64_t B, int64_t Tm, int64_t Nm, hipStream_t stream);

/* replaces: get_segments / get_segments_numpy utils/segments.py:41-72 (callers generator/__init__.py:147-158, base_lightning_module.py:38-44) */
int osp_gather_rows(const float* src, const int64_t* start, int64_t mult, float* out, int64_t B, int64_t T, int64_t S, int64_t C, hipStream_t stream);

/* replaces: expand_by_duration generator/alignments.py:283-297 */
int osp_expand_by_duration(const float* x, const int64_t* dur, float* out, int64_t B, int64_t Nm, int64_t Tout, int64_t C, hipStream_t stream);

/* ---- api.cpp ---- */
/* replaces: error text of the last failing call on this thread */
const char* osp_last_error();

/* replaces: measurement aid, no reference counterpart: symbol and algorithmic flops of the matrix-core kernel(s) the calling thread's last entry-point call launched (bench.py's roofline block reads it; cleared by the read) */
int osp_kernel_note_host(char* name_host, int64_t cap, double* flops_host);

/* replaces: measurement aid: algorithmic HBM bytes of the launches osp_kernel_note_host reports (decides matrix-pipe-bound vs HBM-bound) */
int osp_kernel_note_bytes_host(double* bytes_host);

/* replaces: ABI version of this library */
int osp_abi_version();

/* replaces: content hash of the sources this library was built from (optispeech_amd/build.py checks it; no reference counterpart) */
const char* osp_source_hash();

/* replaces: torch.cuda.Event.record + Stream.wait_event of the multi-stream schedule in one call (no reference counterpart: the reference runs on one stream) */
int osp_stream_handover(void* event_host_handle, void* dst_stream_host_handle, hipStream_t stream);

/* replaces: no reference counterpart: zero / byte fill of a buffer inside a taped region (torch.zeros / Tensor.zero_ of the host code) */
int osp_memset(void* dst, int64_t value, int64_t nbytes, hipStream_t stream);

/* replaces: no reference counterpart: device-to-device copy inside a taped region (torch.cat / Tensor.copy_ of the host code) */
int osp_copy(void* dst, const void* src, int64_t nbytes, hipStream_t stream);

/* replaces: test aid of the call tapes: adds into a HOST counter, no device work (lets the CPU suite record / patch / replay) */
int osp_tape_selftest(int64_t* counter, int64_t add, hipStream_t stream);

/* replaces: test aid of the call tapes: sums host int64 values addressed through a host table (copy + patching of descriptor tables) */
int osp_tape_selftest_table(const int64_t* vals_host, int64_t count, int64_t* counter, hipStream_t stream);

/* ---- attention.hip ---- */
/* replaces: MultiHeadedAttention.forward_attention masked softmax + dropout: generator/modules/_transformer/attention.py:75-97 */
int osp_attn_softmax_fwd(float* S, float* Pd, const int64_t* klen, int64_t B, int64_t H, int64_t T1, int64_t T2, float scale, float drop_p, int64_t seed, const int64_t* seed_dev, int64_t stream_id, hipStream_t stream);

/* replaces: autograd of the same (softmax' and the dropout mask regenerated from the Philox counter) */
int osp_attn_softmax_bwd(const float* P, float* dPd, int64_t rows, int64_t T2, float scale, float drop_p, int64_t seed, const int64_t* seed_dev, int64_t stream_id, hipStream_t stream);

/* replaces: MultiHeadedAttention.forward_attention without the (T x T) scores in HBM (no-grad / inference path): _transformer/attention.py:75-101 */
int osp_attn_fused_fwd(const float* q, const float* k, const float* v, const int64_t* klen, float* o, int64_t B, int64_t H, int64_t T, int64_t DK, float scale, hipStream_t stream);

/* ---- attention_packed_bwd.hip ---- */
/* replaces: workspace query for osp_packed_attention_bwd */
int64_t osp_packed_attention_bwd_workspace_bytes(int64_t docs, int64_t qlongest, int64_t Mk, int64_t Hq, int64_t Hk, int64_t D, int64_t bf16);

/* replaces: autograd of the same: probabilities recomputed per tile from q, k and the log-sum-exp */
int osp_packed_attention_bwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const void* o, const void* rest, const float* lse, const void* dout, int64_t do_row, int64_t do_head, int64_t bf16, void* dq, void* dk, void* dv, float* delta, void* workspace, const int64_t* qbegin, const int64_t* qlen, const int32_t* qtiles, const int32_t* qntiles, int64_t qcap, const int64_t* kbegin, const int64_t* klen, const int32_t* ktiles, const int32_t* kntiles, int64_t kcap, const int64_t* prefix, const float* slopes, int64_t docs, int64_t qlongest, int64_t klongest, int64_t Mq, int64_t Mk, int64_t Hq, int64_t Hk, int64_t D, float scale, float softcap, int64_t causal, hipStream_t stream);

/* ---- attention_packed_fwd.hip ---- */
/* replaces: MultiHeadedAttention.forward_attention on packed documents, with capped scores, a penalty on distance, causal and prefix masks, shared key heads and different query / key counts (generator/modules/_transformer/attention.py:75-125 knows a key-padding mask) */
int osp_packed_attention_fwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int64_t bf16, void* o, void* rest, float* lse, const int64_t* qlen, const int32_t* qtiles, const int32_t* qntiles, int64_t qcap, const int64_t* kbegin, const int64_t* klen, const int64_t* prefix, const float* slopes, int64_t docs, int64_t klongest, int64_t Mq, int64_t Hq, int64_t Hk, int64_t D, float scale, float softcap, int64_t causal, hipStream_t stream);

/* ---- attention_packed_token.hip ---- */
/* replaces: workspace query for osp_packed_attention_token */
int64_t osp_packed_attention_token_workspace_bytes(int64_t B, int64_t Mq, int64_t longest, int64_t Hq, int64_t Hk, int64_t D);

/* replaces: osp_packed_attention_fwd for few queries over many keys (new frames over a cache): keys split over workgroups and joined */
int osp_packed_attention_token(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int64_t bf16, void* o, void* workspace, const int64_t* qbegin, const int64_t* qlen, const int32_t* qtiles, const int32_t* qntiles, int64_t qcap, const int64_t* kbegin, const int64_t* klen, int64_t longest, const int64_t* prefix, const float* slopes, int64_t B, int64_t Mq, int64_t Hq, int64_t Hk, int64_t D, float scale, float softcap, int64_t causal, hipStream_t stream);

/* ---- attention_train.hip ---- */
/* replaces: MultiHeadedAttention.forward scores -> masked softmax -> dropout -> P V in ONE kernel (training): generator/modules/_transformer/attention.py:80-98,120-125; keeps the per-row log-sum-exp only */
int osp_attn_train_fwd(const float* q, const float* k, const float* v, const int64_t* klen, const float* sbias, float* o, float* lse, int64_t B, int64_t H, int64_t T, int64_t DK, float scale, float drop_p, int64_t seed, const int64_t* seed_dev, int64_t stream_id, hipStream_t stream);

/* replaces: autograd of the same: probabilities recomputed per tile from q, k and the log-sum-exp (no (T x T) tensor) */
int osp_attn_train_bwd(const float* q, const float* k, const float* v, const float* o, const float* lse, const float* dout, const int64_t* klen, const float* sbias, float* dsbias, float* dq, float* dk, float* dv, float* Dbuf, int64_t B, int64_t H, int64_t T, int64_t DK, float scale, float drop_p, int64_t seed, const int64_t* seed_dev, int64_t stream_id, hipStream_t stream);

/* ---- comm.cpp ---- */
/* replaces: rendezvous id of the gradient communicator (Lightning DDP strategy setup, configs/trainer/ddp.yaml:4-9) */
int osp_comm_unique_id(void* id_host);

/* replaces: DDP process-group construction for the gradient all-reduce (configs/trainer/ddp.yaml:4-9) */
int osp_comm_init(int64_t rank, int64_t world, const void* id_host);

/* replaces: number of ranks of the initialised communicator (0 = none) */
int64_t osp_comm_world();

/* replaces: DDP's bucketed gradient all-reduce (torch.nn.parallel.DistributedDataParallel reducer behind manual_backward, base_lightning_module.py:99,119) */
int osp_allreduce_bucket(float* ptr, int64_t n, hipStream_t stream);

/* replaces: process-group teardown */
int osp_comm_destroy();

/* ---- convnext.hip ---- */
/* replaces: ConvNeXtBlock.forward dwconv + LayerNorm: generator/modules/convnext.py:36-38 */
int osp_dwconv7_ln_fwd(const float* x, const float* dw, const float* dwb, const float* lnw, const float* lnb, float eps, void* h, int64_t h_bf16, float* xhat, float* rstd, int64_t B, int64_t T, int64_t C, hipStream_t stream);

/* replaces: nn.LayerNorm: convnext.py:85,102; modules/layers.py:26-45 (eps 1e-12) + nn.Dropout core.py:74; wavenext/__init__.py:84 */
int osp_layernorm_fwd(const float* x, const float* w, const float* b, float eps, float* y, float* mean, float* rstd, const float* rowmask, float drop_p, int64_t seed, const int64_t* seed_dev, int64_t stream_id, int64_t rows, int64_t C, hipStream_t stream);

/* replaces: autograd of the LayerNorm (+ReLU, +Dropout) call sites above */
int osp_layernorm_bwd(const float* dy, const float* xin, const float* mean, const float* rstd, const float* w, const float* relu_src, const float* rowmask, float drop_p, int64_t seed, const int64_t* seed_dev, int64_t stream_id, float* dx, float* dlnw, float* dlnb, int64_t rows, int64_t C, float* ws, int64_t ws_blocks, hipStream_t stream);

/* replaces: autograd of nn.Conv1d(groups=dim) at generator/modules/convnext.py:36 */
int osp_dwconv7_bwd(const float* dc, const float* x, const float* dw, const float* dres, const float* dres_rowmask, float* dx, float* ddw, float* ddb, int64_t B, int64_t T, int64_t C, hipStream_t stream);

/* replaces: autograd of LayerNorm + depthwise Conv1d(k=7) of ConvNeXtBlock in one pass: generator/modules/convnext.py:36-38 (C <= 256) */
int osp_ln_dwconv7_bwd(const float* dh, const float* xhat, const float* rstd, const float* lnw, const float* x, const float* dw, const float* dres, const float* dres_rowmask, float* dx, float* dlnw, float* dlnb, float* ddw, float* ddb, int64_t B, int64_t T, int64_t C, float* ws, int64_t ws_blocks, hipStream_t stream);

/* ---- dwconv.hip ---- */
/* replaces: depthwise nn.Conv1d(groups = C, odd k) and its input gradient (flip = 1): ConvSeparable modules/layers.py:455-477, _conformer/convolution.py */
int osp_dwconv_fwd(const float* x, const float* w, const float* bias, const float* rowmask, float* y, int64_t B, int64_t T, int64_t C, int64_t K, int64_t flip, hipStream_t stream);

/* replaces: autograd weight / bias gradient of the same depthwise Conv1d */
int osp_dwconv_wgrad(const float* dy, const float* x, const float* rowmask, float* dw, float* db, int64_t B, int64_t T, int64_t C, int64_t K, hipStream_t stream);

/* replaces: F.dropout (+ residual add) call sites of the separable-conv layers: modules/layers.py:497-503; backward = the same kernel on the gradient */
int osp_dropout_add(const float* x, const float* res, float* y, int64_t n, float p, int64_t seed, const int64_t* seed_dev, int64_t stream_id, hipStream_t stream);

/* ---- embed.hip ---- */
/* replaces: TextEmbedding.forward modules/core.py:25-31, ScaledSinusoidalEmbedding modules/layers.py:48-71 */
int osp_text_embed_fwd(const int64_t* tok, const float* E, const float* pos, const float* scale, float sqrt_dim, float drop_p, int64_t seed, const int64_t* seed_dev, int64_t stream_id, float* out, int64_t B, int64_t T, int64_t C, hipStream_t stream);

/* replaces: autograd of nn.Embedding(padding_idx=0) + ScaledSinusoidalEmbedding.scale */
int osp_text_embed_bwd(const float* dy, const int64_t* tok, const float* pos, float sqrt_dim, float drop_p, int64_t seed, const int64_t* seed_dev, int64_t stream_id, int64_t padding_idx, float* dE, float* dscale, int64_t B, int64_t T, int64_t C, hipStream_t stream);

/* ---- ew.hip ---- */
/* replaces: no reference counterpart: the per-step dropout seed written to device memory (kernels read it through seed_dev) */
int osp_store_i64(int64_t* dst, int64_t value, hipStream_t stream);

/* replaces: autograd's gradient accumulation (a tensor with several consumers), negation and scalar scaling inside taped regions */
int osp_ew_axpby(const float* x, const float* y, float* out, int64_t n, float a, float b, hipStream_t stream);

/* replaces: element-wise products with a row / column broadcast: `x * mask` sites of modules/core.py:161-175 and their autograd */
int osp_ew_mul(const float* x, const float* y, float* out, int64_t n, int64_t inner, int64_t mode, hipStream_t stream);

/* replaces: autograd of the scalar loss assembly: gradient tensor times an incoming device scalar (generator/loss.py, alignments.py:236-238) */
int osp_ew_scale_dev(const float* x, const float* s, float* out, int64_t n, float c, hipStream_t stream);

/* replaces: autograd of nn.ReLU after nn.Conv1d: modules/core.py:66-71 */
int osp_ew_relu_mask(const float* g, const float* y, float* out, int64_t n, hipStream_t stream);

/* replaces: mel.transpose(1, 2) of OptiSpeechGenerator.forward: generator/__init__.py:122 */
int osp_transpose_last2(const float* x, float* y, int64_t B, int64_t R, int64_t C, hipStream_t stream);

/* replaces: sequence_mask + padding masks: utils/model.py:12-16, generator/__init__.py:96-103 */
int osp_length_masks(const int64_t* len, int64_t B, int64_t T, float* keep, void* pad_bool, hipStream_t stream);

/* replaces: torch.mean over the per-utterance loss terms: generator/loss.py:190-193, alignments.py:236-238 */
int osp_sum_scaled(const float* x, int64_t n, float scale, float* out, hipStream_t stream);

/* replaces: weighted loss sums: generator/__init__.py:175-181, vocoder/wavenext/disc/__init__.py:105-111 */
int osp_dot_multi(const int64_t* x_host, const float* coeff_host, int64_t count, float* out, float* terms, hipStream_t stream);

/* replaces: autograd of the weighted loss sums */
int osp_scale_vec(const float* g, const float* coeff_host, int64_t count, float* out, hipStream_t stream);

/* replaces: ScaledPositionalEncoding.forward `x + alpha * pe`: generator/modules/_transformer/embedding.py:120-124 */
int osp_posenc_fwd(const float* x, const float* pe, const float* alpha, float* y, int64_t B, int64_t n, hipStream_t stream);

/* replaces: autograd of the same w.r.t. alpha (stage 1: one partial per workgroup; stage 2 = osp_sum_scaled) */
int osp_posenc_dalpha(const float* dy, const float* pe, int64_t B, int64_t n, float* partials, int64_t nparts, hipStream_t stream);

/* replaces: the head split / merge `.view(B, T, h, d_k).transpose(1, 2)` (+ .contiguous()) of MultiHeadedAttention: generator/modules/_transformer/attention.py:59-66,99-101 */
int osp_permute_0213(const float* x, float* y, int64_t A, int64_t B, int64_t C, int64_t D, hipStream_t stream);

/* ---- fused_small.hip ---- */
/* replaces: FeatureMatchingLoss.forward over ALL feature-map pairs of a discriminator family in one launch: disc/loss.py:68-85 */
int osp_l1_sum_multi(const int64_t* a_host, const int64_t* b_host, const int64_t* n_host, const float* scale_host, const int64_t* bf16_host, int64_t count, float* out, hipStream_t stream);

/* replaces: autograd of the same */
int osp_l1_sign_multi(const int64_t* a_host, const int64_t* b_host, const int64_t* gb_host, const int64_t* n_host, const float* scale_host, const int64_t* bf16_host, int64_t count, const float* gscale, hipStream_t stream);

/* replaces: GeneratorLoss / DiscriminatorLoss hinge terms of all sub-discriminators in one launch: disc/loss.py:11-65 */
int osp_hinge_sum_multi(const int64_t* x_host, const int64_t* n_host, const float* sgn_host, const float* scale_host, int64_t count, float* out, hipStream_t stream);

/* replaces: autograd of the same */
int osp_hinge_grad_multi(const int64_t* x_host, const int64_t* dx_host, const int64_t* n_host, const float* sgn_host, const float* scale_host, int64_t count, const float* gscale, hipStream_t stream);

/* replaces: torch.nn.utils.weight_norm forward of many convs in one launch (see osp_wnorm_fwd) */
int osp_wnorm_fwd_multi(const int64_t* desc_host, int64_t count, hipStream_t stream);

/* replaces: autograd of weight_norm for many convs in one launch (see osp_wnorm_bwd) */
int osp_wnorm_bwd_multi(const int64_t* desc_host, int64_t count, hipStream_t stream);

/* replaces: autograd of the layer scale `self.gamma * x`: ConvNeXtBlock.forward generator/modules/convnext.py:45-46 */
int osp_colsum_prod(const float* a, const float* b, const float* rowf, float* out, int64_t M, int64_t C, hipStream_t stream);

/* replaces: no reference counterpart: row-scaled f32 -> bf16 operand copy (drop-path / mask factor folded in) */
int osp_cast_bf16_rows(const float* x, const float* rowscale, void* y, int64_t M, int64_t C, hipStream_t stream);

/* replaces: SpectralConvergenceLoss + LogSTFTMagnitudeLoss reductions (torch.norm / F.l1_loss of log magnitudes) and the mel L1: disc/loss.py:107-120,231-270 */
int osp_spectral_loss_sums(const float* x, const float* y, int64_t n, float clip, float* sums, hipStream_t stream);

/* replaces: autograd of the same with respect to the predicted magnitudes */
int osp_spectral_loss_bwd(const float* x, const float* y, int64_t n, float clip, const float* sums, const float* g, float* dx, hipStream_t stream);

/* replaces: get_random_segments start indices: utils/segments.py:12-38 (caller generator/__init__.py:147-153) */
int osp_segment_starts(const float* r01, const int64_t* lens, int64_t B, int64_t lead, int64_t segment_size, int64_t* out, hipStream_t stream);

/* replaces: DropPath factors of all blocks of a ConvNeXt backbone: generator/modules/convnext.py:121-129 (drop_p_host: plain host array) */
int osp_drop_path_rows(const float* drop_p_host, const float* rowmask, int64_t L, int64_t B, int64_t T, int64_t seed, const int64_t* seed_dev, int64_t stream_id, float* scale, float* rowf, hipStream_t stream);

/* replaces: DiscriminatorP.forward reflect pad + (b, t/p, p) view as period-column sequences, and its gradient (backward = 1): vocoder/wavenext/disc/_discriminators.py:63-72 */
int osp_period_fold(const float* x, float* y, int64_t B, int64_t T, int64_t period, int64_t backward, hipStream_t stream);

/* replaces: torch.clip(audio, -1, 1) of WaveNeXtHead.forward and its backward: vocoder/wavenext/__init__.py:47 */
int osp_clip(const float* x, const float* dy, float* out, int64_t n, float lo, float hi, hipStream_t stream);

/* ---- gemm.hip ---- */
/* replaces: nn.Linear / nn.Conv1d forward + dgrad: generator/modules/convnext.py:39-41, modules/core.py:66-71,95, generator/alignments.py:55-64, vocoder/wavenext/__init__.py:43-44,83; torch.matmul in alignments.py:173 */
int osp_conv_gemm_f32(const float* A, int64_t lda, int64_t M, int64_t T, int64_t Cin, int64_t taps, int64_t pad, const float* a_rowscale, const float* B, int64_t sBn, int64_t sBtap, int64_t sBk, int64_t N, float* C, int64_t ldc, int64_t epi, const float* bias, const float* gamma, const float* res, int64_t ldr, const float* rowmask, const float* rowscale, float* aux_out, const float* aux_in, int64_t ld_aux, int64_t batch, int64_t sAb, int64_t sBb, int64_t sCb, int64_t sXb, int64_t accumulate, hipStream_t stream);

/* replaces: autograd weight/bias gradients of the same nn.Linear / nn.Conv1d call sites */
int osp_conv_wgrad_f32(const float* dY, int64_t ldy, const float* X, int64_t ldx, int64_t M, int64_t T, int64_t N, int64_t Cin, int64_t taps, int64_t pad, const float* arow, const float* oscale, float* dW, int64_t ldw, float* db, int64_t batch, int64_t sYb, int64_t sXb, int64_t sWb, int64_t sDb, hipStream_t stream);

/* ---- gemm_bf16.hip ---- */
/* replaces: same call sites as osp_conv_gemm_f32 and the weight-normed Conv2d (k,1) stacks of DiscriminatorP (vocoder/wavenext/disc/_discriminators.py:51-60,80-90), bf16 operands / f32 accumulate */
int osp_conv_gemm_bf16(const void* A, int64_t a_bf16, int64_t lda, int64_t M, int64_t Trows, int64_t Tin, int64_t Cin, int64_t taps, int64_t a_step, int64_t a_tapstep, int64_t a_off, const float* a_rowscale, const void* B, int64_t b_bf16, int64_t sBn, int64_t sBtap, int64_t sBk, int64_t N, void* C, int64_t c_bf16, int64_t ldc, int64_t Tc, int64_t c_step, int64_t c_off, int64_t epi, const float* bias, const float* gamma, const void* res, int64_t res_bf16, int64_t ldr, const float* rowmask, const float* rowscale, void* aux_out, const void* aux_in, int64_t aux_bf16, int64_t ld_aux, float slope, int64_t batch, int64_t sAb, int64_t sBb, int64_t sCb, int64_t sXb, int64_t accumulate, hipStream_t stream);

/* replaces: weight-normed Conv2d forward of DiscriminatorP / DiscriminatorR + F.leaky_relu: vocoder/wavenext/disc/_discriminators.py:51-60,63-97 and :154-163,165-194 */
int osp_conv2d_gemm_bf16(const void* A, int64_t a_bf16, int64_t lda, int64_t M, int64_t Trows, int64_t Wrows, int64_t Hin, int64_t Win, int64_t Cin, int64_t taps, int64_t KW, int64_t a_step_h, int64_t a_tapstep_h, int64_t a_off_h, int64_t a_step, int64_t a_tapstep, int64_t a_off, const void* B, int64_t b_bf16, int64_t sBn, int64_t sBtap_h, int64_t sBtap, int64_t sBk, int64_t N, void* C, int64_t c_bf16, int64_t ldc, int64_t Tc, int64_t Wc, int64_t c_step_h, int64_t c_off_h, int64_t c_step, int64_t c_off, int64_t epi, const float* bias, const void* res, int64_t res_bf16, int64_t ldr, const void* aux_in, int64_t aux_bf16, int64_t ld_aux, float slope, hipStream_t stream);

/* replaces: autograd input gradients of the same strided Conv2d stacks (all stride phases in one launch) */
int osp_conv2d_dgrad_bf16(const void* dy, int64_t dy_bf16, const void* wt, int64_t w_bf16, void* dx, int64_t dx_bf16, int64_t U, int64_t H, int64_t W, int64_t Ho, int64_t Wo, int64_t Cin, int64_t Cout, int64_t KH, int64_t KW, int64_t sh, int64_t sw, int64_t ph, int64_t pw, int64_t epi, const void* aux_in, int64_t aux_bf16, const void* res, int64_t res_bf16, float slope, hipStream_t stream);

/* ---- gemm_f32_glds.hip ---- */
/* replaces: same call sites as osp_conv_gemm_f32 (f32 operands in HBM), products as three bf16 MFMAs over (hi, lo) operand pairs: the 'mixed' parity mode's generator GEMMs outside the index-critical path */
int osp_conv_gemm_f32_split(const float* A, int64_t lda, int64_t M, int64_t T, int64_t Cin, int64_t taps, int64_t pad, const float* a_rowscale, const float* B, int64_t sBn, int64_t sBtap, int64_t sBk, int64_t N, float* C, int64_t ldc, int64_t epi, const float* bias, const float* gamma, const float* res, int64_t ldr, const float* rowmask, const float* rowscale, float* aux_out, const float* aux_in, int64_t ld_aux, int64_t batch, int64_t sAb, int64_t sBb, int64_t sCb, int64_t sXb, int64_t accumulate, hipStream_t stream);

/* ---- group_norm.hip ---- */
/* replaces: workspace query for osp_group_norm_fwd / osp_group_norm_bwd */
int64_t osp_group_norm_workspace_bytes(int64_t B, int64_t M, int64_t C, int64_t G, int64_t backward);

/* replaces: no reference counterpart: group norm + activation over the rows of each document (the place of BatchNorm + swish in _conformer/convolution.py:61-70, which counts padded frames); stats: (3, B, G) f32, mean, 1 / deviation and the mean's part below f32 */
int osp_group_norm_fwd(const void* x, int64_t ldx, int64_t bf16, const float* w, const float* b, void* y, float* stats, void* workspace, const int64_t* begin, const int64_t* len, const int32_t* base, const int32_t* tiles, const int32_t* ntiles, int64_t cap, int64_t B, int64_t M, int64_t longest, int64_t C, int64_t G, float eps, int64_t act, hipStream_t stream);

/* replaces: autograd of the same */
int osp_group_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t bf16, const float* w, const float* b, const float* stats, void* dx, float* dw, int64_t add_w, float* db, int64_t add_b, void* workspace, const int64_t* begin, const int64_t* len, const int32_t* base, const int32_t* tiles, const int32_t* ntiles, int64_t cap, int64_t B, int64_t M, int64_t longest, int64_t C, int64_t G, int64_t act, hipStream_t stream);

/* ---- loss.hip ---- */
/* replaces: FastSpeech2Loss.forward generator/loss.py:83-140, DurationPredictorLoss :28-46 */
int osp_variance_losses(const float* d_hat, const float* p_hat, const float* e_hat, const float* ds, const float* ps, const float* es, const int64_t* x_len, float clip_val, float* out, float* gd, float* gp, float* ge, int64_t B, int64_t T, hipStream_t stream);

/* replaces: workspace query for osp_forwardsum_ctc */
int64_t osp_forwardsum_ctc_workspace_floats(int64_t B, int64_t Tm, int64_t Nm);

/* replaces: ForwardSumLoss.forward generator/loss.py:150-194 (F.log_softmax + F.ctc_loss per item) and its autograd */
int osp_forwardsum_ctc(const float* lp, const int64_t* x_len, const int64_t* y_len, float blank_logprob, float* workspace, float* loss_item, float* grad, int64_t B, int64_t Tm, int64_t Nm, hipStream_t stream);

/* ---- lstm.hip ---- */
/* replaces: recurrence of nn.LSTM(dim, dim, 1, batch_first=True) after the input-projection GEMM: generator/modules/leanspeech.py:49-60 (hx / flags: workspace, flags zeroed) */
int osp_lstm_fwd(const float* gx, const float* whh, float* hs, float* gates, float* cs, float* hx, int32_t* flags, int64_t B, int64_t T, int64_t H, hipStream_t stream);

/* replaces: autograd of the same recurrence: gradient w.r.t. the gate pre-activations for every step (dW / db / dx are GEMMs over it) */
int osp_lstm_bwd(const float* dhs, const float* gates, const float* cs, const float* whh, float* dg, int32_t* flags, int64_t B, int64_t T, int64_t H, hipStream_t stream);

/* ---- mlp_fused.hip ---- */
/* replaces: no reference counterpart: bf16 weight pack of pwconv2 in the k order osp_convnext_mlp_fused reads it in */
int osp_pack_bf16_kperm16(const float* w, void* out, int64_t N, int64_t K, hipStream_t stream);

/* replaces: the same, walking the rows in a given order (unmasked rows first) with the caller's count of unmasked rows (synthesise knows the sum of the utterance lengths after its one length sync, generator/__init__.py:258-262): masked row blocks leave at once */
int osp_convnext_mlp_fused_live(const void* h, const void* w1, const float* b1, const void* w2_kperm, const float* b2, const float* gamma, const float* x, const float* rowmask, const float* rowscale, float* y, int64_t M, int64_t C, int64_t I, const int* rowperm, int64_t live_rows, hipStream_t stream);

/* replaces: ConvNeXtBlock.forward pwconv1 -> GELU -> pwconv2 -> gamma, residual (+ backbone mask) without gradients, hidden activations never in HBM: generator/modules/convnext.py:39-46,99-101 (callers: OptiSpeechGenerator.synthesise generator/__init__.py:170-228, WaveNeXt.forward vocoder/wavenext/__init__.py:77-88) */
int osp_convnext_mlp_fused(const void* h, const void* w1, const float* b1, const void* w2_kperm, const float* b2, const float* gamma, const float* x, const float* rowmask, const float* rowscale, float* y, int64_t M, int64_t C, int64_t I, hipStream_t stream);

/* replaces: no reference counterpart: the rows of a padded batch in the order 'unmasked first' (a stable partition by the padding mask), which osp_convnext_mlp_fused_live walks */
int osp_row_order(const float* rowmask, int* perm, int64_t M, hipStream_t stream);

/* ---- optim.hip ---- */
/* replaces: clip_grad_norm_ total norm (LightningModule.clip_gradients, base_lightning_module.py:100-102,120-122) */
int osp_sumsq(const float* g, int64_t n, double* out, hipStream_t stream);

/* replaces: torch.optim.AdamW.step + clip_gradients: base_lightning_module.py:96-105,116-125; configs/model/optimizer/adamw.yaml */
int osp_adamw_clip(float* p, const float* g, float* m, float* v, int64_t n, const double* sumsq, const float* lr_dev, const int64_t* step_dev, float lr, float beta1, float beta2, float eps, float wd, int64_t step, float max_norm, float gscale, hipStream_t stream);

/* ---- packed_rows.hip ---- */
/* replaces: no reference counterpart: most tiles the tile list of a packed batch can have (the reference pads every batch) */
int64_t osp_packed_rows_tiles(int64_t B, int64_t M);

/* replaces: no reference counterpart: documents and tile list of a packed or padded batch, from offsets / lengths on the device */
int osp_packed_rows_plan(const int64_t* src, int64_t padded, int64_t B, int64_t M, int64_t T, int64_t* begin, int64_t* len, int32_t* base, int32_t* tiles, int32_t* ntiles, int64_t cap, hipStream_t stream);

/* ---- rotary.hip ---- */
/* replaces: no reference counterpart: rotary positions of q and k per document, forward and backward (the reference adds sinusoids or uses relative positions: generator/modules/_transformer/embedding.py:91-124,252-322) */
int osp_rotary(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, int64_t in_bf16, void* qo, void* ko, int64_t out_bf16, const double* turns, const int32_t* tiles, const int32_t* ntiles, int64_t cap, const int64_t* first, int64_t Hq, int64_t Hk, int64_t D, int64_t R, int64_t interleaved, float mag, int64_t inverse, hipStream_t stream);

/* ---- smallcin.hip ---- */
/* replaces: first layers Conv2d(1, 32, (k,1)) / Conv2d(1, 32, (7,5)) and the 32-channel DiscriminatorR layers: disc/_discriminators.py:53,156-160 */
int osp_smallcin_conv_fwd(const float* x, const float* w, const float* b, void* y, int64_t y_bf16, int64_t M, int64_t Trows, int64_t Wrows, int64_t Hin, int64_t Win, int64_t Cout, int64_t taps, int64_t KW, int64_t sh, int64_t sw, int64_t ph, int64_t pw, int64_t lrelu, float slope, hipStream_t stream);

/* replaces: autograd weight/bias gradients of the same narrow-channel layers */
int osp_smallcin_conv_wgrad(const float* x, const void* dy, int64_t y_bf16, float* dw, float* db, int64_t M, int64_t Trows, int64_t Wrows, int64_t Hin, int64_t Win, int64_t Cout, int64_t taps, int64_t KW, int64_t sh, int64_t sw, int64_t ph, int64_t pw, float* ws, int64_t ws_floats, hipStream_t stream);

/* ---- stft.hip ---- */
/* replaces: twiddle table for the STFT kernels (torch.stft internals) */
int osp_fft_twiddles(float* tw, int64_t N, hipStream_t stream);

/* replaces: torch.stft(...).abs(): disc/loss.py:123-142, disc/_discriminators.py:196-216, torchaudio MelSpectrogram disc/loss.py:94-107 */
int osp_stft_mag_fwd(const float* x, const float* window, const float* tw, float clamp_min, float* mag, int64_t B, int64_t T, int64_t N, int64_t hop, hipStream_t stream);

/* replaces: autograd of the same */
int osp_stft_mag_bwd(const float* x, const float* window, const float* tw, float clamp_min, const float* dmag, float* dx, int64_t B, int64_t T, int64_t N, int64_t hop, hipStream_t stream);

/* replaces: CommonFeatureExtractor.get_mel mel_basis @ magnitudes + spectral_normalize_torch, and get_energy's torch.norm: dataset/feature_extractors/__init__.py:143-146,197-199; utils/audio.py:23-24 */
int osp_logmel_energy(const float* mag, const float* fbT, float* mel_out, float* energy_out, int64_t F, int64_t bins, int64_t n_mels, float eps, float clip, hipStream_t stream);

/* ---- wgrad_bf16.hip ---- */
/* replaces: weight gradients of the same, bf16 operands / f32 accumulate */
int osp_conv_wgrad_bf16(const void* dY, int64_t y_bf16, int64_t ldy, const void* X, int64_t x_bf16, int64_t ldx, int64_t M, int64_t Trows, int64_t Tin, int64_t N, int64_t Cin, int64_t taps, int64_t pad, int64_t x_step, const float* arow, const float* oscale, float* dW, int64_t ldw, float* db, int64_t batch, int64_t sYb, int64_t sXb, int64_t sWb, int64_t sDb, hipStream_t stream);

/* replaces: the same weight gradients with a caller-supplied split workspace: no f32 atomics, bit-reproducible (autograd of nn.Conv1d / nn.Linear: generator/modules/convnext.py:39-41) */
int osp_conv_wgrad_bf16_ws(const void* dY, int64_t y_bf16, int64_t ldy, const void* X, int64_t x_bf16, int64_t ldx, int64_t M, int64_t Trows, int64_t Tin, int64_t N, int64_t Cin, int64_t taps, int64_t pad, int64_t x_step, const float* arow, const float* oscale, float* dW, int64_t ldw, float* db, int64_t batch, int64_t sYb, int64_t sXb, int64_t sWb, int64_t sDb, float* ws, int64_t ws_bytes, hipStream_t stream);

/* replaces: autograd weight gradients of the same Conv2d stacks */
int osp_conv2d_wgrad_bf16(const void* dY, int64_t y_bf16, int64_t ldy, const void* X, int64_t x_bf16, int64_t ldx, int64_t M, int64_t Trows, int64_t Wrows, int64_t Hin, int64_t Win, int64_t N, int64_t Cin, int64_t taps, int64_t KW, int64_t pad_h, int64_t pad, int64_t x_step_h, int64_t x_step, float* dW, float* db, hipStream_t stream);

/* replaces: autograd weight gradients of the DiscriminatorP / DiscriminatorR Conv2d stacks (vocoder/wavenext/disc/_discriminators.py:51-60,154-163) with a split workspace instead of atomics */
int osp_conv2d_wgrad_bf16_ws(const void* dY, int64_t y_bf16, int64_t ldy, const void* X, int64_t x_bf16, int64_t ldx, int64_t M, int64_t Trows, int64_t Wrows, int64_t Hin, int64_t Win, int64_t N, int64_t Cin, int64_t taps, int64_t KW, int64_t pad_h, int64_t pad, int64_t x_step_h, int64_t x_step, float* dW, float* db, float* ws, int64_t ws_bytes, hipStream_t stream);

/* replaces: no reference counterpart: f32 -> bf16 operand copy for the MFMA kernels (the reference's autocast does this implicitly) */
int osp_cast_bf16(const float* x, void* y, int64_t n, hipStream_t stream);

/* replaces: no reference counterpart: (Cout, Cin, K) -> tap-major bf16 weight layout for the conv-GEMM kernels */
int osp_pack_bf16(const float* w, const float* kscale, void* out, int64_t N, int64_t taps, int64_t K, int64_t sN, int64_t sT, int64_t sK, hipStream_t stream);

/* replaces: no reference counterpart: osp_pack_bf16 for a list of weights in one launch */
int osp_pack_bf16_multi(const int64_t* desc_host, int64_t count, hipStream_t stream);

/* ---- wgrad_ring.hip ---- */
/* replaces: exact-f32 weight gradients (the f32 / mixed parity modes) with a split workspace: no f32 atomics (autograd of nn.Conv1d / nn.Linear: generator/modules/convnext.py:39-41, generator/alignments.py:55-64) */
int osp_conv_wgrad_f32_ws(const float* dY, int64_t ldy, const float* X, int64_t ldx, int64_t M, int64_t T, int64_t N, int64_t Cin, int64_t taps, int64_t pad, const float* arow, const float* oscale, float* dW, int64_t ldw, float* db, int64_t batch, int64_t sYb, int64_t sXb, int64_t sWb, int64_t sDb, float* ws, int64_t ws_bytes, hipStream_t stream);

/* replaces: the same weight gradients (f32 operands in HBM) with products as three bf16 MFMAs over (hi, lo) operand pairs: the 'mixed' parity mode's generator */
int osp_conv_wgrad_f32_split_ws(const float* dY, int64_t ldy, const float* X, int64_t ldx, int64_t M, int64_t T, int64_t N, int64_t Cin, int64_t taps, int64_t pad, const float* arow, const float* oscale, float* dW, int64_t ldw, float* db, int64_t batch, int64_t sYb, int64_t sXb, int64_t sWb, int64_t sDb, float* ws, int64_t ws_bytes, hipStream_t stream);

/* ---- wnorm.hip ---- */
/* replaces: torch.nn.utils.weight_norm forward w = g * v / ||v|| at every DiscriminatorP/R conv: disc/_discriminators.py:7,53-60,156-163 */
int osp_wnorm_fwd(const float* v, const float* g, void* wn_bf16, float* wn_f32, void* wt_bf16, float* inv_norm, int64_t Cout, int64_t Cin, int64_t P, int64_t Q, hipStream_t stream);

/* replaces: autograd of weight_norm: gradients of weight_g / weight_v from the effective-weight gradient */
int osp_wnorm_bwd(const float* dwn, const float* v, const float* g, const float* inv_norm, float* dv, float* dg, int64_t Cout, int64_t Cin, int64_t P, int64_t Q, hipStream_t stream);

/* replaces: FeatureMatchingLoss.forward torch.mean(torch.abs(rl - gl)): disc/loss.py:68-85 */
int osp_l1_sum(const void* a, const void* b, int64_t is_bf16, int64_t n, float scale, float* out, hipStream_t stream);

/* replaces: autograd of the same */
int osp_l1_sign(const void* a, const void* b, int64_t is_bf16, int64_t n, float scale, const float* gscale, void* gb, hipStream_t stream);

/* replaces: GeneratorLoss / DiscriminatorLoss hinge terms mean(clamp(1 -/+ d, min=0)): disc/loss.py:11-65 */
int osp_hinge_sum(const float* x, int64_t n, float sgn, float scale, float* out, hipStream_t stream);

/* replaces: autograd of the same */
int osp_hinge_grad(const float* x, int64_t n, float sgn, float scale, const float* gscale, float* dx, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* OSP_H */
