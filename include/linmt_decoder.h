/* linmt_decoder.h -- C ABI of the B200 beam-search decoding engine.
 *
 * The library replaces LiNMT's sentence-decoding path.  Every entry point takes plain
 * pointers and sizes; nothing here depends on a tensor library.  Unless a function says
 * otherwise, pointers are HOST pointers and the call copies to and from the GPU itself.
 *
 * Citations are into the reference project's tree (src/...).
 */
#ifndef LINMT_DECODER_H_
#define LINMT_DECODER_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------------------
 * 1. The reference's own exported symbols (src/decoder_sentence.h:94-97, definitions
 *    src/decoder_sentence.cu:847-873).  Same names, same signatures, same ownership rule:
 *    the returned string belongs to the library and stays valid until the next call.
 *    `msg` is the path of a decoding-sentence config file (param="--key" value="..." lines,
 *    src/decoder_sentence.cu:267-318).  Like the reference, init prints and exits the
 *    process on a fatal configuration error; do_job never exits and returns "" on error.
 * ------------------------------------------------------------------------------------ */
void python_decoder_init(char* msg);
char* python_decoder_do_job(char* sentence);

/* UNK post-processing, the pair the reference's wrapper and server call right after
 * python_decoder_do_job (src/postprocess_unks.h:89-92, definitions src/postprocess_unks.cc:716-752;
 * callers server/LiNMT-python-wrapper.py:24-33, server/LiNMT-server.py:52-57).  Host string code.
 * `msg` = config file with --phrase-table ("src ||| tgt ||| x" lines), --stopword and --end-punct
 * (tab-separated "tag<TAB>word" lines) and optional --rm-oov-mode; init exits on a missing file as
 * the reference does.  do_job takes the source line (optionally "words |||| {generalizations}") and
 * the decoder's "words |||| score |||| alignments |||| unk alignments |||| a/a/a ..." line and
 * returns the final words; the string belongs to the library until the next call. */
void python_unk_init(char* msg);
char* python_unk_do_job(char* src_sentence, char* translation);
/* The same on a handle, returning the whole line with its "||||" fields
 * (PostProcessUnks::Init / Process, src/postprocess_unks.cc:14-30). */
typedef struct linmt_unk linmt_unk;
int linmt_unk_create(const char* config_path, linmt_unk** out);
int linmt_unk_process(const linmt_unk* h, const char* source, const char* translation, char* out, int32_t out_cap);
void linmt_unk_destroy(linmt_unk* h);

/* ------------------------------------------------------------------------------------
 * 2. Handle-based API at the reference's numeric boundary
 *    (EnsembleFactory<T>::InitDecoderSentence, src/decoder.h:1526-1575, and
 *    EnsembleFactory<T>::DecodeSentence, src/decoder.h:1780-1840), extended from one
 *    sentence per call to a batch of independent sentences.
 * ------------------------------------------------------------------------------------ */
typedef struct linmt_engine linmt_engine;

enum { LINMT_OK = 0, LINMT_EINVAL = 1, LINMT_ECUDA = 2, LINMT_EIO = 3, LINMT_ENOMEM = 4, LINMT_ELIMIT = 5 };

enum { LINMT_ATT_LOCAL_P_GENERAL = 0, LINMT_ATT_GLOBAL_GENERAL = 1, LINMT_ATT_GLOBAL_DOT = 2 };
enum { LINMT_ENS_PROB_MEAN = 0, LINMT_ENS_LOGPROB_MEAN = 1 };
enum { LINMT_PREC_FP32 = 0, LINMT_PREC_BF16 = 1 };
/* GEMM kernel family.  SIMT = fp32 CUDA-core kernels (fp32 FMA arithmetic).  TENSOR = tcgen05
 * tensor-core kernels; with fp32 precision every operand is held as an fp16 pair x ~ a0 + 2^-11 a1
 * (22 mantissa bits, three partial products per product, fp32-class accuracy; operands must be
 * below 65504 in magnitude).  TENSOR3 = three bf16 planes (six partial products, same accuracy,
 * no range limit), TENSOR2 = two bf16 planes (error ~2^-17 per product).  TENSOR_V16 = TENSOR for the
 * recurrent and attention products, but the vocabulary projection in plain fp16 (one product instead of three:
 * logits carry ~2^-12 relative noise, 1e-5 on a log-probability; near-ties in the beam may resolve differently;
 * ~15 % faster).  TENSOR_V16X = TENSOR_V16 plus a refinement in the softmax kernel: every logit that can still
 * be among the k+1 best of its row given the error bound of the fp16 product (and EOS) is recomputed from both
 * planes, so candidates and their log-probabilities are fp32-class again; only the normaliser sums fp16 logits.
 * AUTO = TENSOR_V16X for a single model (measured: the same parity as TENSOR, 13 % faster), TENSOR for ensembles. */
enum { LINMT_GEMM_AUTO = 0, LINMT_GEMM_SIMT = 1, LINMT_GEMM_TENSOR = 2, LINMT_GEMM_TENSOR2 = 3, LINMT_GEMM_TENSOR3 = 4, LINMT_GEMM_TENSOR_V16 = 5, LINMT_GEMM_TENSOR_V16X = 6 };

/* Model dimensions: first five of the nine integers on line 1 of a model file
 * (src/decoder.h:1202-1210). */
typedef struct linmt_model_desc {
  int32_t layers;      /* L  */
  int32_t hidden;      /* H = LSTM size = embedding size */
  int32_t vocab_tgt;   /* V  */
  int32_t vocab_src;   /* Vs */
  int32_t feed_input;  /* 1 = previous attentional state feeds layer 1 */
} linmt_model_desc;

/* Decoding options; defaults are the reference's (src/global_configuration.h:228-235). */
typedef struct linmt_options {
  int32_t beam;            /* 12; clamped to floor(sqrt(V)) (src/decoder.h:1549-1551)      */
  int32_t nbest;           /* 1                                                            */
  int32_t attention_mode;  /* LINMT_ATT_*                                                  */
  int32_t attention_d;     /* local attention half width D, 10 (src/global_configuration.h:45) */
  int32_t print_info;      /* 1 = track viterbi and dense alignments (--print-decoding-info) */
  int32_t precision;       /* LINMT_PREC_*                                                 */
  int32_t ensemble_mode;   /* LINMT_ENS_*                                                  */
  int32_t gemm_path;       /* LINMT_GEMM_*: which hand-written GEMM kernel family to use   */
  int32_t max_batch;       /* most sentences per device batch (64)                         */
  int32_t max_src_len;     /* longest source sentence accepted (100)                       */
  int32_t max_steps;       /* most beam expansions per sentence (200)                      */
  int32_t device;          /* CUDA device ordinal                                          */
  float penalty;           /* 0    */
  float diversity;         /* 0    */
  float lp_alpha;          /* 0.65 */
  float cp_beta;           /* 0.20 */
  float min_ratio;         /* 0.5: keep hypotheses with len/S > min_ratio (src/decoder.h:762-765) */
  float max_ratio;         /* 1.5: only used by the sentence API to derive the step count
                              min((int)(max_ratio*S), longest-2) (src/decoder.h:1806)      */
} linmt_options;

/* Fills `opt` with the defaults above. */
void linmt_default_options(linmt_options* opt);

/* Number of floats in one weight blob of the given shape. */
size_t linmt_blob_floats(const linmt_model_desc* desc);

/* Creates an engine from in-memory weights.  `blobs[m]` is ensemble member m: the matrices
 * of a model file in LoadWeights order (src/deep_rnn.h:1878-1969), each rows x cols
 * column-major as the reference holds them on the device (src/deep_rnn_kernel.h:1543-1560).
 * Replaces DecoderModelWrapper::InitDecoderSentence + LoadWeights
 * (src/decoder.h:1040-1107, src/deep_rnn.h:1878-1969). */
int linmt_create_from_weights(const linmt_model_desc* desc, const float* const* blobs, int32_t n_models,
                              size_t blob_floats, const linmt_options* opt, linmt_engine** out);

/* The same engine on several GPUs of one box: devices[0..n_devices) each get a replica of the model(s)
 * (opt->device is then ignored), and linmt_decode_batch / linmt_decode_file deal device batches of
 * sentences to them, one host thread per device inside the library; nothing crosses between the GPUs
 * and results come back in the caller's order.  Sentences are independent in the reference too
 * (EnsembleFactory::DecodeSentence keeps no state between calls, src/decoder.h:1780-1840); its own use
 * of several GPUs is one DecoderModelWrapper per GPU index (src/decoder.h:1676-1684, config key
 * --multi-gpu, src/decoder_sentence.cu:183-198), which this replaces.  n_devices = 0 means opt->device. */
int linmt_create_from_weights_on(const linmt_model_desc* desc, const float* const* blobs, int32_t n_models,
                                 size_t blob_floats, const linmt_options* opt, const int32_t* devices,
                                 int32_t n_devices, linmt_engine** out);
/* Number of devices a handle decodes on. */
int32_t linmt_device_count(const linmt_engine* e);

/* Creates an engine from a decoding-sentence config file, reading the model file(s) named
 * by --nmt-model in the reference's text format.  Replaces DecoderSentence::Init
 * (src/decoder_sentence.cu:14-37). */
int linmt_create(const char* config_path, linmt_engine** out);

void linmt_destroy(linmt_engine* e);

/* Text of the last error on this handle (or of the last failed create when e == NULL).
 * A decode that returns LINMT_ECUDA with "gave up waiting on a barrier" leaves the handle unusable:
 * every wait inside the GEMM kernels is bounded (about a second) and a wait that ran out means the
 * device state of this handle can no longer be trusted, so every later decode on it fails the same
 * way.  Destroy the handle and create a new one. */
const char* linmt_last_error(const linmt_engine* e);
/* Text of the last error of linmt_create / linmt_read_model_file (config and model-file problems). */
const char* linmt_front_error(void);

/* Effective beam after clamping. */
int32_t linmt_beam(const linmt_engine* e);

/* Optional per-step records of a decode, and optional forcing of the beam.
 * All pointers are host pointers and may be NULL.  Tm = max steps[i], k = effective beam.
 *   cand_tok, cand_logp   [n][Tm][k][k+1]  per-beam top-(k+1) tokens and log-probabilities
 *   surv_tok, surv_parent, surv_score [n][Tm][k]  survivors chosen at each step
 *   final_logp            [n][k]  log p(EOS) at the extra forward
 *   force_tok, force_parent, force_score [n][Tm][k]  if set, the beam continues from these
 *                         survivors instead of its own (the records still show its own). */
typedef struct linmt_trace {
  int32_t* cand_tok;
  float* cand_logp;
  int32_t* surv_tok;
  int32_t* surv_parent;
  float* surv_score;
  float* final_logp;
  const int32_t* force_tok;
  const int32_t* force_parent;
  const float* force_score;
  float* gold_logp;   /* [n][Tm][k]: log p of the forced token of each slot (needs force_*), may be NULL */
  float* pt;          /* [n_models][n][Tm+1][k]: attention centre p_t of every forward of every ensemble member (local
                         attention), may be NULL.  Entries of forwards that did not run hold the bit pattern 0xffffffff. */
} linmt_trace;

/* Decodes n independent sentences.  Replaces EnsembleFactory<T>::DecodeSentence
 * (src/decoder.h:1780-1840) and Decoder<T>::ObtainOneBestHypothesis (src/decoder.h:703-859)
 * up to, not including, the formatting of the output string.
 *   src_ids, src_off  sentence i = src_ids[src_off[i] .. src_off[i+1]) in natural order
 *                     (the engine reverses it as src/decoder_sentence.cu:68 does)
 *   steps             T_i beam expansions for sentence i; one more forward appends EOS
 *   max_len           row length of the outputs, >= max T_i + 2
 *   out_tok   [n][nbest][max_len]  hypothesis including START(0) and EOS(1)
 *   out_len   [n][nbest]           its length, 0 = fewer than nbest hypotheses passed the filter
 *   out_score [n][nbest]
 *   out_vit   [n][nbest][max_len]  viterbi alignment per position, may be NULL
 *   out_align [n][nbest][max_len][max_src_len]  dense alignments, may be NULL (print_info only)
 * Sentences are processed in device batches of at most max_batch.  A call of a single model that has several device batches of up to
 * 512 beam slots runs two or three of them at once on every device (linmt_score_batch, in batches of up to 512 sentences, and
 * linmt_decode_file do the same), each on an engine with the handle's weights and state of its own:
 *   - One or two further engines per device are made by the first such call, beside its first batches, and kept until the
 *     handle is destroyed.  That call is up to 1.5 ms longer than without them, later ones are shorter (64 sentences a batch,
 *     4 x 1000 / 30k: 300 greedily 46.5 ms one after another, 34 to 36 the first call, 32 after it).
 *   - An engine takes 0.1 (2 x 128, greedily) to 0.7 GB of device memory (4 x 1000 / 30k, beam 12), and 0.2 GB more where it
 *     scores.  None is made that takes more than 3 GB or a quarter of what the device has free, and a call that is refused memory
 *     gives them up and runs on the handle's own engines.
 *   - In fp32 precision the products of batches that share a device add in another order: the last bits of a score (4e-7 of it)
 *     go by whether the call has one device batch or several that run at once.  Repeated calls give the same bits.  bf16
 *     results do not depend on it. */
int linmt_decode_batch(linmt_engine* e, const int32_t* src_ids, const int32_t* src_off, int32_t n,
                       const int32_t* steps, int32_t max_len, int32_t* out_tok, int32_t* out_len,
                       float* out_score, int32_t* out_vit, float* out_align, const linmt_trace* trace);

/* Same decode with every buffer already in device memory (no host copies inside): the
 * sentences must fit one device batch (n <= max_batch), `steps` is still a host array
 * because it sizes the launches.  Outputs stay on the device. */
int linmt_decode_batch_device(linmt_engine* e, const int32_t* d_src_ids, const int32_t* src_off_host,
                              int32_t n, const int32_t* steps_host, int32_t max_len, int32_t* d_out_tok,
                              int32_t* d_out_len, float* d_out_score);

/* Counters since creation: kernels launched by this library, decoder forwards (row-steps)
 * and device time of the last decode call in milliseconds (CUDA events). */
typedef struct linmt_stats {
  int64_t kernel_launches;
  int64_t decoder_row_steps;
  int64_t sentence_steps;
  float last_decode_ms;
  float last_gemm_ms;     /* time inside the dominant (vocabulary) GEMM launches, if timing is on */
  int32_t last_gemm_launches;
  int32_t last_rec_gemm_launches; /* decoder LSTM-stack GEMM launches of the last call, if timing is on */
  float last_rec_gemm_ms;         /* time inside them */
  float last_host_issue_ms;       /* host time spent issuing the decoder steps of the last device batch */
  double last_rec_gemm_flops;     /* their algorithmic flops: 2 * rows * 4H * K per launch */
  int64_t pair_launches;          /* GEMM launches, of kernel_launches, that ran on CTA pairs (tcgen05 cta_group::2) */
} linmt_stats;
int linmt_get_stats(const linmt_engine* e, linmt_stats* out);
/* 1 = put a CUDA event before every kernel of the decoder steps (for roofline measurements).  The events
 * end the overlap of consecutive kernels, so a timed decode is a measurement pass: slower than an untimed one. */
int linmt_set_kernel_timing(linmt_engine* e, int32_t on);
/* Device time and launch count per kernel class of the last timed device batch (first device of the handle).
 * Classes in launch order: 0 state gather, 1 LSTM gate GEMMs, 2 attention projections GEMM, 3 attention,
 * 4 attention output GEMM (no launches on the tensor-core path: that layer is applied to the encoder states once per
 * batch and finished inside the attention kernel), 5 vocabulary GEMM, 6 ensemble combination (with its softmax), 7 softmax / top-k, 8 beam
 * selection (no launches: it runs inside 6 and 7).  `ms` and `launches` hold n >= 9 entries. */
int linmt_kernel_times(const linmt_engine* e, float* ms, int32_t* launches, int32_t n);

/* Sentence API on a handle: DecoderSentence::Process (src/decoder_sentence.cu:40-49).
 * Needs an engine created from a config file (vocabularies).  Returns a library-owned
 * string valid until the next call on the same handle. */
const char* linmt_translate(linmt_engine* e, const char* sentence);

/* Force-decoding / scoring: log-probability of given target sentences under the model
 * (the reference's --force-decoding path, src/deep_rnn.h:1490-1568, src/dispatcher.cu:699-752).
 *   tgt_ids, tgt_off  target token ids per sentence WITHOUT START / EOS
 *   out_logprob [n]   sum over the m_i tokens and the closing EOS of log p(token | source, prefix)
 *   out_token_logp    optional [n][max_tgt + 1]: the per-token terms (EOS last), zero padded
 * Every sentence needs 1 <= m_i <= max_steps.  Several device batches run at once: see linmt_decode_batch. */
int linmt_score_batch(linmt_engine* e, const int32_t* src_ids, const int32_t* src_off, const int32_t* tgt_ids,
                      const int32_t* tgt_off, int32_t n, float* out_logprob, float* out_token_logp, int32_t max_tgt);

/* Reads a model file in the reference's text format (header, vocabularies, matrices; the format
 * written by DumpBestModel, src/deep_rnn.h:1972-2146, and read by LoadWeights, :1878-1969) without
 * creating an engine: fills `desc` and, if `blob` is given, the weights in the blob layout of
 * linmt_create_from_weights (`blob_cap` floats available).  use_cache = 1 reads / writes the raw
 * copy "<path>.linmtcache" that makes later loads of the same unchanged text file fast.  No GPU call. */
int linmt_read_model_file(const char* path, linmt_model_desc* desc, float* blob, uint64_t blob_cap, int32_t use_cache);

/* File-mode decoding: one source sentence per line of `in_path`; writes the n-best
 * translations of every sentence to `out_path` in input order.  Replaces
 * EnsembleFactory::DecodeFile (src/decoder.h:1702-1776), Decoder::OutputKBestHypotheses
 * (src/decoder.h:529-699) and InputFilePreprocess::UnintFile
 * (src/input_file_preprocess.cc:1485-1572).  Needs an engine created from a config file; sentences
 * are decoded in length-sorted batches of --batch-size, several at once: see linmt_decode_batch. */
int linmt_decode_file(linmt_engine* e, const char* in_path, const char* out_path);

/* ------------------------------------------------------------------------------------
 * 3. Single-kernel entry points (host pointers) used by the parity tests.
 * ------------------------------------------------------------------------------------ */
/* Y[R][N] = X[R][K] . W[K][N] with W stored like a reference weight ([in][out]);
 * stands in for one cublasSgemm call of the reference (src/utility_cu.h:153-157).
 * gemm_path: LINMT_GEMM_SIMT or LINMT_GEMM_TENSOR; precision: LINMT_PREC_*. */
int linmt_k_gemm(const float* X, const float* W, float* Y, int32_t R, int32_t K, int32_t N, int32_t gemm_path,
                 int32_t precision, int32_t device);
/* The vocabulary product of a step as the engine runs it, and the softmax behind it: Y = X[R][K] . W[K][V] + bias, the
 * statistics that the product leaves per block of columns, and every row's top-kk log-probabilities.
 *   gemm_path   LINMT_GEMM_AUTO (fp32: one fp16 product, the values rounded to fp16, the candidates recomputed) or
 *               LINMT_GEMM_TENSOR (fp32: three products); LINMT_PREC_BF16: one bf16 product either way
 *   block_max, block_sum  [R][ld], ld = 4 * ceil(Vp / 48) + 4, Vp = V rounded up to 128: maximum of a block and sum of
 *               exp(value - maximum) over it.  Block i covers columns [c, c + info[3]) of tile i / 4, c = (i % 4) * info[3],
 *               as far as the tile (info[2] columns) and V go
 *   info [5]    kernel that ran (0 one tile per CTA, 1 few rows, 2 CTA pairs, 3 persistent, 4 persistent pairs), blocks,
 *               columns of a tile and of a block, 1 if the sums were left too */
int linmt_k_logits(const float* X, const float* W, const float* bias, int32_t R, int32_t K, int32_t V, int32_t gemm_path, int32_t precision, int32_t kk,
                   float* Y, float* block_max, float* block_sum, int32_t* info, int32_t* idx, float* logp, float* eos_logp, int32_t device);
/* Per-row log-softmax statistics and top-kk of logits[R][V]: replaces the softmax kernel
 * (src/deep_rnn_kernel.h:352-429) plus the per-beam top-(k+1) scan of
 * src/decoder.h:401-410.  idx/logp are [R][kk], eos_logp [R]. */
int linmt_k_softmax_topk(const float* logits, int32_t R, int32_t V, int32_t kk, int32_t* idx, float* logp,
                         float* eos_logp, int32_t device);

/* What linmt_attend_pages8 leaves where its kernel gives up a wait: in this thread's calls from now on every `each`-th CTA does so before its first one (0: none, as at the start). */
int linmt_k_attend8_give_up(int32_t each);

/* Y[R][N] = X[R][K] . Wt[N][K]^T on the tensor-core kernel (three bf16 planes, fp32-class
 * result) WITHOUT allocating: for hosts that cannot call cudaMalloc once they are running --
 * processes that gave the whole GPU to their own memory pool at start-up, or that share the
 * device and must not trigger the device-wide stall an allocation can cause.  It has no
 * counterpart in the reference.
 *   d_x, d_wt, d_y  DEVICE pointers, fp32, row-major; K a multiple of 32, N a multiple of 16.
 *   Limits: R <= 256, K <= 1024, N <= 1024 (LINMT_ELIMIT beyond): the kernel's working memory
 *   (the bf16 planes of both operands, 7.5 MiB) is a fixed array inside the library that every
 *   GPU loading the library holds until exit.
 * The first call on a device looks that array's address up (cudaGetSymbolAddress); make it
 * before any stream capture.  Work is issued on the default stream and the call returns when
 * the result is in d_y.  All calls share the one array and it keeps the last call's contents:
 * two calls that overlap on the GPU (from two threads, say) race -- serialise them. */
int linmt_gemm_f32_noalloc(const float* d_x, const float* d_wt, float* d_y, int32_t R, int32_t K, int32_t N,
                           int32_t device);

/* ------------------------------------------------------------------------------------
 * 4. Operators on device tensors, for programs that run their own model and want a decoding step's
 *    parts: beam selection and reordering, pages for a growing memory, keys and values in them in
 *    4 or 8 bits, attention over them, pages that follow their hypotheses, scores of given tokens.  They have no counterpart in the reference, whose beam search runs on the
 *    host (src/decoder.h:340-525) and whose attention reads dense states.
 *
 *    Every pointer inside the argument structs is a DEVICE pointer on `device`, every stride is in elements unless
 *    it says bytes.  A call checks its arguments, issues its kernels on `stream` (a cudaStream_t, NULL = the default
 *    stream) and returns without waiting; nothing is allocated and nothing is kept between calls, so calls may run at once
 *    and may be captured into a graph, as long as their outputs and workspaces are not shared.  The current device is left as it
 *    was.  LINMT_EINVAL: an argument is not allowed; LINMT_ELIMIT: a size is beyond what the kernel is made for;
 *    LINMT_ECUDA: the launch was refused; linmt_op_error() has the text, per host thread.  `size` is sizeof the struct.
 * ------------------------------------------------------------------------------------ */
enum { LINMT_F32 = 0, LINMT_BF16 = 1, LINMT_F16 = 2 };

const char* linmt_op_error(void);

/* Beam selection: of the k * vocab continuations of each sentence's beams the k best, best first.
 *   a live beam b      offers every word v with score_b + x_v - log sum_u exp(x_u) over its allowed logits x
 *   a finished beam    offers `eos` alone, with its score as it is; its logits are not read
 *   a beam whose score is not finite, and one with a NaN or +inf at an allowed place, offers nothing
 * Equal sums go to the lowest b * vocab + v.  The order is that of 64-bit arithmetic as far as 2^-36: sums of two beams that lie closer
 * than 32 bits can tell apart are compared again with normalisers that are good to that.  Words that are not allowed may hold anything;
 * one whose logit is -inf is never chosen.  Slots that nothing is left for get token eos, parent = the slot itself, score -inf, done 1.
 * out_scores and out_done may be the arrays `scores` and `done`; nothing else that is written may overlap what is read. */
typedef struct linmt_beam_select_args {
  uint32_t size;
  int32_t device;
  void* stream;
  const void* logits;        /* [n][k][vocab], LINMT_F32 / BF16 / F16, words contiguous, aligned to their type */
  int64_t stride_n, stride_k;
  const float* scores;       /* [n][k] */
  const uint8_t* done;       /* [n][k], not 0 = finished; may be NULL */
  const uint32_t* allowed;   /* bit v % 32 of word v / 32 set = word v allowed, ceil(vocab / 32) words; may be NULL */
  int64_t allowed_stride;    /* words from one sentence's list to the next, 0 = one list for all */
  int32_t* out_tokens;       /* [n][k] */
  int32_t* out_parents;      /* [n][k], 0 .. k-1 */
  float* out_scores;         /* [n][k] */
  uint8_t* out_done;         /* [n][k]: parent was finished, or the token is eos */
  int32_t n, k, vocab, eos, dtype;   /* k <= 32, k * vocab <= 2^31 - 4096 */
} linmt_beam_select_args;
int linmt_beam_select(const linmt_beam_select_args* args);

/* Rows of states follow their beams: dst[l][i][j] = src[l][i][parents[i][j]] for every state, one launch for up to 16 of them.
 * dst may be src (the same pointer and strides); otherwise the two must not overlap, nor may a dst and another state.  A parent outside 0 .. k-1 takes the row's own. */
typedef struct linmt_beam_state {
  const void* src;
  void* dst;
  int64_t src_stride_l, src_stride_n, src_stride_k;   /* bytes */
  int64_t dst_stride_l, dst_stride_n, dst_stride_k;
  int64_t row_bytes;
  int64_t layers;
} linmt_beam_state;
typedef struct linmt_beam_reorder_args {
  uint32_t size;
  int32_t device;
  void* stream;
  const int32_t* parents;    /* [n][k] */
  int32_t n, k;              /* k <= 32 */
  int32_t n_states, reserved;
  linmt_beam_state state[16];
} linmt_beam_reorder_args;
int linmt_beam_reorder(const linmt_beam_reorder_args* args);

/* Pages for sentences that grow from old_len to new_len positions: every page column p of sentence i with
 * ceil(old / page) <= p < ceil(new / page) gets the next entry of `free_pages`, sentence by sentence, and every new position its
 * slot = table[i][pos / page] * page + pos % page, sentence by sentence.  Lengths are taken as 0 .. width * page, a shorter new length as the
 * old one.  Where the free list has run out a column gets -1; a position in a column that holds none of the pool's pages gets slot -1;
 * so do slots behind the last new position.  out_used = used + the pages that were wanted (more than n_free: the list ran out).
 * Nothing that is written, the table among it, may overlap the lengths, the free pages or `used`. */
typedef struct linmt_plan_pages_args {
  uint32_t size;
  int32_t device;
  void* stream;
  const int32_t* old_len;    /* [n]; NULL = all 0 */
  const int32_t* new_len;    /* [n] */
  int32_t* table;            /* [n][width], rows `table_stride` apart */
  int64_t table_stride;
  const int32_t* free_pages; /* [n_free] */
  const int32_t* used;       /* [1]: entries of free_pages that are taken already */
  int32_t* out_used;         /* [1], not the array `used` */
  int64_t* out_slots;        /* [total] */
  int32_t* out_starts;       /* [n + 1]: first new position of each sentence in out_slots */
  int32_t n, width, page, n_free;    /* n <= 16384 */
  int64_t total;
} linmt_plan_pages_args;
int linmt_plan_pages(const linmt_plan_pages_args* args);

/* A pool of pages in 4 bits: [n_pages][heads][page / 16] tiles of 18 * dim bytes (dim 64 or 128, page a multiple of 16), 16-byte
 * aligned.  A tile holds 16 positions of one head:
 *   8 dim bytes of key codes (4 bits, low half of a byte first): the codes of components 32 g + 8 c .. + 7 of position t are the
 *     32-bit word t * dim / 8 + c * dim / 32 + g
 *   dim bytes of key scales: bf16 [16][dim / 32]
 *   8 dim bytes of value codes: 16-byte unit (i * 8 + g) * 4 + c has, as 16-bit fours of codes [2][2][2], for position
 *     8 a + 2 c + b and components 64 i + 32 h + 4 g .. + 3 the four [a][h][b]
 *   dim bytes of value scales: bf16 [16][dim / 32]
 * A code stands for (code - 8) * scale.  scale = bf16(m / -8), m the component of largest size of the 32 (the positive one of two);
 * code = 8 + x / scale rounded to the nearest even integer and held to -8 .. 7, computed in 32 bits; scale 0: code 8.  NaN is
 * taken as 0, larger sizes as the largest finite bf16. */
typedef struct linmt_pages4 {
  void* data;
  int64_t stride_page, stride_head;   /* bytes, multiples of 16; the tiles of a page's head are contiguous */
  int32_t n_pages, heads, page, dim;
} linmt_pages4;

/* Keys and values of `t` positions into (write) or out of (read) the slots of a pool.  A slot outside 0 .. n_pages * page - 1 is not written, and reads
 * as zeros.  Slots of a write must differ: what two writes of one slot leave there is not defined.  What is written overlaps nothing that is read. */
typedef struct linmt_pages4_rows_args {
  uint32_t size;
  int32_t device;
  void* stream;
  linmt_pages4 pages;
  const int64_t* slots;      /* [t] */
  void* k;                   /* [t][heads][dim], components contiguous; 16-byte aligned rows */
  void* v;
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;
  int32_t t, dtype;
} linmt_pages4_rows_args;
int linmt_write_pages4(const linmt_pages4_rows_args* args);
int linmt_read_pages4(const linmt_pages4_rows_args* args);

/* Attention of g query rows per sentence (its beams) over the sentence's positions in a pool.  Query head h reads head
 * h / (heads / pages.heads) of the pool; position t of sentence i is row t % page of page table[i][t / page].
 *   s = scale * q . k_t;  cap > 0: s = cap * tanh(s / cap);  slope: s -= slope[h] * |t - centre[i][row]|
 *   seen: first[i][row] <= t < last[i][row] (NULL: all), 0 <= t < len[i], and the table names a page of the pool
 *   out = sum over seen of softmax(s) * v_t; lse = log sum over seen of exp(s).  Nothing seen: 0 and -inf.  A query with a NaN or an infinity that
 *   sees something: NaN and NaN (and so may one above 1e33 in size, whose scores leave 32 bits on the way).
 * `len` beyond width * page is taken as that.  Sums are held in 32 bits.  Weights times scales are
 * rounded to fp16, with a power of 2 for each row that follows the largest of them (2^-97 to 2^99): to 2^-11 of each, or 2^-21 of the row's largest so far; for 32-bit queries,
 * which are multiplied as two fp16 terms, they are two such terms too: 2^-22, or 2^-31.  With 16-bit queries the matrix unit cuts the sums off at some 2^-13 of the weighted
 * mean of a component's scales (2^-16 of its group's largest).  With 16-bit queries a cap is good to 3e-7 of itself up to 64, to 2^-21 of a score above.
 * `workspace`: linmt_attend_pages4_workspace bytes, 16-byte aligned, the call's own until it has run; NULL where that is 0. */
typedef struct linmt_attend_pages4_args {
  uint32_t size;
  int32_t device;
  void* stream;
  linmt_pages4 pages;
  const void* q;             /* [n][g][heads][dim], components contiguous, rows 4-byte aligned */
  int64_t q_stride_n, q_stride_g, q_stride_h;
  void* out;                 /* as q, strides of its own; q itself with q's strides, or apart from it; apart from all else that is read */
  int64_t out_stride_n, out_stride_g, out_stride_h;
  float* lse;                /* [n][g][heads]; may be NULL */
  const int32_t* table;      /* [n][width], rows `table_stride` apart */
  int64_t table_stride;
  const int32_t* len;        /* [n] */
  const float* slope;        /* [heads]; may be NULL */
  const float* centre;       /* [n][g]; with slope */
  const int32_t* first;      /* [n][g]; may be NULL */
  const int32_t* last;       /* [n][g]; with first */
  void* workspace;
  int64_t workspace_bytes;
  int32_t n, g, heads, width, dtype;
  float scale, cap;
} linmt_attend_pages4_args;
int64_t linmt_attend_pages4_workspace(const linmt_attend_pages4_args* args);   /* bytes, or -1: see linmt_op_error */
int linmt_attend_pages4(const linmt_attend_pages4_args* args);

/* A pool of pages in 8 bits: [n_pages][heads][page / 16] blocks of 32 * dim + 16 bytes (dim 64 or 128, page a multiple of 16), 16-byte
 * aligned.  A block holds 16 positions of one head:
 *   16 dim bytes of key codes: position t, component c is byte (t / 8) * 8 dim + (c / 16) * 128 + (t % 8) * 16 + c % 16
 *   16 dim bytes of value codes: byte 16 c + t
 *   the keys' scale and the values' scale, float, and 8 bytes of zeros
 * A code is a signed byte, -127 .. 127, and stands for code * scale.  A scale is 4, 5, 6 or 7 times a power of 2, 2^-126 at least, or 0. */
typedef struct linmt_pages8 {
  void* data;
  int64_t stride_page, stride_head;   /* bytes, multiples of 16; the blocks of a page's head are contiguous */
  int32_t n_pages, heads, page, dim;
} linmt_pages8;

/* Keys and values of `t` positions into (write) or out of (read) the slots of a pool.  A slot outside 0 .. n_pages * page - 1 is not written, and reads
 * as zeros.  A write goes by runs: neighbours in `slots` that are neighbours in a block, ascending, as linmt_plan_pages gives them.
 *   A run that begins at a block's first position makes the block new: its scale is the run's.  One that begins further on keeps the
 *   positions before it, and the block's scale if it reaches the run's; otherwise the run's becomes the block's and earlier codes are rounded to it: c = code * old / new.
 *   Positions of the block behind the run become zeros.
 *   The run's scale is the smallest whose 127-fold reaches its largest component in size, of the keys and the values each; code = component /
 *   scale, a quotient in 32 bits rounded to the nearest integer, to even between two.  NaN is taken as 0, sizes above 2^127 as 2^127.  Scale 0: code 0.
 * What two runs of one call in the same block leave there is not defined.  What is written overlaps nothing that is read. */
typedef struct linmt_pages8_rows_args {
  uint32_t size;
  int32_t device;
  void* stream;
  linmt_pages8 pages;
  const int64_t* slots;      /* [t] */
  void* k;                   /* [t][heads][dim], components contiguous; 16-byte aligned rows */
  void* v;
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;
  int32_t t, dtype;
} linmt_pages8_rows_args;
int linmt_write_pages8(const linmt_pages8_rows_args* args);
int linmt_read_pages8(const linmt_pages8_rows_args* args);

/* Attention of g query rows per sentence over the sentence's positions in a pool of 8-bit pages, as linmt_attend_pages4 with one argument more:
 *   seen: t < sinks or first[i][row] <= t < last[i][row] (NULL: all), 0 <= t < len[i], and the table names a page of the pool
 * A query's components are taken to 2^-22 of its row's largest (of 2^-106 for smaller ones); their products with the codes are summed exactly, and so are those of the weights:
 * a weight times its block's scale is taken to 2^-30 of the row's largest, with 16-bit queries to 2^-27.  Scores are held in 32 bits.  With 16-bit queries a cap of up to 64 is good to 3e-7 of itself.
 * A query with a NaN or an infinity that sees something: NaN and NaN; so may one whose scores leave 32 bits.  All waits inside the kernel are bounded: rows of a CTA that gave up are NaN. */
typedef struct linmt_attend_pages8_args {
  uint32_t size;
  int32_t device;
  void* stream;
  linmt_pages8 pages;
  const void* q;             /* [n][g][heads][dim], components contiguous, aligned to their type */
  int64_t q_stride_n, q_stride_g, q_stride_h;
  void* out;                 /* as q, strides of its own; q itself with q's strides, or apart from it; apart from all else that is read */
  int64_t out_stride_n, out_stride_g, out_stride_h;
  float* lse;                /* [n][g][heads]; may be NULL */
  const int32_t* table;      /* [n][width], rows `table_stride` apart */
  int64_t table_stride;
  const int32_t* len;        /* [n] */
  const float* slope;        /* [heads]; may be NULL */
  const float* centre;       /* [n][g]; with slope */
  const int32_t* first;      /* [n][g]; may be NULL */
  const int32_t* last;       /* [n][g]; with first */
  void* workspace;
  int64_t workspace_bytes;
  int32_t n, g, heads, width, dtype, sinks;   /* sinks >= 0; without `first` all positions are seen anyway */
  float scale, cap;
} linmt_attend_pages8_args;
int64_t linmt_attend_pages8_workspace(const linmt_attend_pages8_args* args);   /* bytes, or -1: see linmt_op_error */
int linmt_attend_pages8(const linmt_attend_pages8_args* args);

/* Pages follow their hypotheses: row r = i * k + j of the new table is row i * k + parents[i][j] of the old one (parents NULL: row r itself); a parent outside
 * 0 .. k-1, or done[i][j], leaves it without pages.  A row names ceil(len / page) pages, lengths taken as 0 .. width * page.
 *   shares[p]   how many rows beyond the first name page p: 0 for a page of one row, and for a free one, as linmt_plan_pages hands them out
 *   a last page that is not full stays with its row's first child; every further child names a page of its own instead, and the page to copy from and
 *               the new one are the next entries of out_src and out_dst, in the order of the rows (linmt_copy_pages); -1 behind the last
 *   pages that no row names any more go back in front of the free ones, ascending: free_pages[used - freed .. used - 1]; new pages are then taken
 *               from there on.  Where they run out a column and its out_dst are -1 and out_used comes back larger than n_free.
 * `used` is taken as 0 .. n_free.  Columns behind a row's pages, and those that name no page of the pool, come out as -1.  The same page in two columns of a row is not
 * allowed: what becomes of its shares is not defined, though nothing outside the arrays is touched.  out_shares, out_free and out_used may be the arrays
 * shares, free_pages and used; nothing else that is written may overlap what is read, or another result. */
typedef struct linmt_fork_pages_args {
  uint32_t size;
  int32_t device;
  void* stream;
  const int32_t* table;      /* [n * k][width], rows `table_stride` apart */
  int64_t table_stride;
  const int32_t* len;        /* [n * k] */
  const int32_t* parents;    /* [n * k]; may be NULL */
  const uint8_t* done;       /* [n * k]; may be NULL */
  const int32_t* shares;     /* [n_pages] */
  const int32_t* free_pages; /* [n_free] */
  const int32_t* used;       /* [1] */
  int32_t* out_table;        /* [n * k][width], rows `out_table_stride` apart */
  int64_t out_table_stride;
  int32_t* out_len;          /* [n * k] */
  int32_t* out_shares;       /* [n_pages] */
  int32_t* out_free;         /* [n_free] */
  int32_t* out_used;         /* [1] */
  int32_t* out_src;          /* [n * k] */
  int32_t* out_dst;          /* [n * k] */
  int32_t n, k, width, page, n_pages, n_free;   /* n * k <= 16384; n * k * width, n_pages and n_free up to 2^31 - 2^17 - 1 */
} linmt_fork_pages_args;
int linmt_fork_pages(const linmt_fork_pages_args* args);

/* The pages that rows name move to the front of their pool: with U of them, each that lies at U or behind takes the place, in order, of one before U that
 * nothing names: out_src, out_dst (linmt_copy_pages), -1 behind the last.  out_table and out_shares go by the new numbers, out_free is 0, 1, .. n_pages - 1 and out_used U.
 * A row names ceil(len / page) pages, lengths taken as 0 .. width * page; other columns come out as -1, and so do those that name no page of the pool.
 * out_table may be `table` (the same pointer and stride), out_shares may be `shares`; nothing else that is written may overlap what is read, or another result. */
typedef struct linmt_compact_pages_args {
  uint32_t size;
  int32_t device;
  void* stream;
  const int32_t* table;      /* [rows][width], rows `table_stride` apart */
  int64_t table_stride;
  const int32_t* len;        /* [rows] */
  const int32_t* shares;     /* [n_pages] */
  int32_t* out_table;        /* [rows][width], rows `out_table_stride` apart */
  int64_t out_table_stride;
  int32_t* out_shares;       /* [n_pages] */
  int32_t* out_free;         /* [n_pages] */
  int32_t* out_used;         /* [1] */
  int32_t* out_src;          /* [n_pages / 2] */
  int32_t* out_dst;          /* [n_pages / 2] */
  int32_t* workspace;        /* [n_pages], the call's own until it has run */
  int32_t rows, width, page, n_pages;   /* rows * width and n_pages up to 2^31 - 2^17 - 1 */
} linmt_compact_pages_args;
int linmt_compact_pages(const linmt_compact_pages_args* args);

/* Copies of whole pages: page dst[i] of every pool becomes what its page src[i] holds, one launch for up to 16 pools.  Entries with a number outside
 * 0 .. n_pages - 1 copy nothing.  No page may be named twice in dst, or in both: what such entries leave there is not defined. */
typedef struct linmt_page_pool {
  void* data;
  int64_t stride_page;       /* bytes */
  int64_t page_bytes;        /* contiguous */
} linmt_page_pool;
typedef struct linmt_copy_pages_args {
  uint32_t size;
  int32_t device;
  void* stream;
  const int32_t* src;        /* [n] */
  const int32_t* dst;        /* [n] */
  int32_t n, n_pages, n_pools, reserved;
  linmt_page_pool pool[16];
} linmt_copy_pages_args;
int linmt_copy_pages(const linmt_copy_pages_args* args);

/* Scores of given tokens: of every row of logits x over its allowed words, with p = softmax(x),
 *   out_logprob        x_token - log sum exp(x); -inf for a word that is not allowed, 0 for a token outside 0 .. vocab - 1 (a padded place)
 *   out_entropy        - sum p log p
 *   out_top_tokens, out_top_logprobs   the `top` words of the largest logits, equal ones by the lowest number; -1 and -inf where no word with a logit above -inf is left
 * A row with a NaN or +inf at an allowed place: NaN, and -1 for words.  One without a word above -inf: -inf (0 for a padded place), and entropy 0. */
typedef struct linmt_score_tokens_args {
  uint32_t size;
  int32_t device;
  void* stream;
  const void* logits;        /* [n][t][vocab], LINMT_F32 / BF16 / F16, words contiguous, aligned to their type */
  int64_t stride_n, stride_t;
  const int32_t* tokens;     /* [n][t] */
  const uint32_t* allowed;   /* as in linmt_beam_select; may be NULL */
  int64_t allowed_stride;    /* words from one n's list to the next, 0 = one list for all */
  float* out_logprob;        /* [n][t] */
  float* out_entropy;        /* [n][t] */
  int32_t* out_top_tokens;   /* [n][t][top]; with top > 0 */
  float* out_top_logprobs;   /* [n][t][top] */
  int32_t n, t, vocab, top, dtype, reserved;   /* top <= 32, n * t below 2^31, vocab <= 2^31 - 4096 */
} linmt_score_tokens_args;
int linmt_score_tokens(const linmt_score_tokens_args* args);

#ifdef __cplusplus
}
#endif
#endif /* LINMT_DECODER_H_ */
