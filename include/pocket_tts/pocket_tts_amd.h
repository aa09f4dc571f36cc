/*
 * Additive C entry points of the MI355X engine.  Nothing here changes the drop-in surface of
 * pocket_tts_c.h; these calls expose (1) options the reference can only set from C++ or its CLI,
 * (2) a batch ingress for many independent utterances, and (3) one entry point per ONNX Runtime
 * call site of the reference so each network can be checked in isolation.  All buffers are host
 * memory unless stated otherwise; sizes are in elements.  Return value 0 = success, -1 = failure with the message available
 * from pocket_tts_get_last_error(), unless stated otherwise.
 */
#ifndef POCKET_TTS_AMD_H
#define POCKET_TTS_AMD_H

#include "pocket_tts_c.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Full option set of the C++ PocketTTSConfig (include/pocket_tts/pocket_tts.hpp:58-68) plus device
 * placement.  Unlike PocketTTSConfig, temperature is taken literally, so 0 selects the deterministic
 * zero start point of src/pocket_tts.cpp:606-613 (the reference reaches that only through its CLI,
 * src/main.cpp:49-50). */
typedef struct {
    const char* models_dir;      /* NULL: "models/onnx" */
    const char* tokenizer_path;  /* NULL: "models/tokenizer.model"; "" or "none": no tokenizer (id-based calls only) */
    const char* precision;       /* NULL: "int8"; "fp32", "bf16" */
    const char* pack_path;       /* NULL: <models_dir>/pocket_tts.ptts */
    float temperature;
    int lsd_steps;               /* <= 0: 10  */
    int max_frames;              /* <= 0: 500 */
    int frames_after_eos;        /* < 0: 3    */
    int device;                  /* HIP device ordinal */
    int max_text_tokens;         /* <= 0: 512 */
    int has_seed;                /* non-zero: seed the noise generator with `seed` */
    unsigned long long seed;
} PocketTTSConfigEx;

POCKET_TTS_API PocketTTSHandle pocket_tts_create_ex(const PocketTTSConfigEx* config);

/* dims[0..7] = latent_dim, d_model, samples_per_frame, vocab, mimi_dim, sample_rate, lsd_steps, max_frames */
POCKET_TTS_API int pocket_tts_dims(PocketTTSHandle handle, int* dims);

/* pocket_tts_encode_voice (/root/reference/include/pocket_tts/pocket_tts_c.h:63, src/pocket_tts_c.cpp:59-82) over n files in one
   call: host threads decode / resample / attenuate / cut the files while the GPU encodes those already prepared.
   voices_out[i] is what pocket_tts_encode_voice(handle, audio_paths[i]) returns (release with pocket_tts_free_voice);
   on failure (-1, pocket_tts_get_last_error) every voices_out[i] is NULL. */
POCKET_TTS_API int pocket_tts_encode_voices(PocketTTSHandle handle, int n, const char* const* audio_paths, VoiceHandle* voices_out);

/* Voice handle <-> raw conditioning rows [frames][d_model]. */
POCKET_TTS_API VoiceHandle pocket_tts_voice_from_embeddings(const float* embeddings, int frames, int d_model);
POCKET_TTS_API int pocket_tts_voice_frames(VoiceHandle voice);
POCKET_TTS_API const float* pocket_tts_voice_data(VoiceHandle voice);

/* n utterances (any n) through the engine's slot table: up to 64 are in flight on the GPU, each with the offline schedule of
 * src/pocket_tts.cpp:548-657, and a slot whose utterance has stopped is refilled from the rest.
 * results[i] is filled like pocket_tts_generate does; release each with pocket_tts_free_audio. */
POCKET_TTS_API int pocket_tts_generate_batch(PocketTTSHandle handle, int n, const char* const* texts,
                                             const VoiceHandle* voices, AudioResult* results);

/* Same, from token ids (the output of the text pre-step, src/tokenizer.cpp:27-60) and raw conditioning rows.
 * noise[i]: NULL, or [max_frames][latent_dim] start points used instead of the internal generator.
 * latents_out[i]: NULL, or room for max_frames*latent_dim floats; eos_out[i]: NULL or max_frames floats.
 * frames_out[i] receives the frame count, eos_count_out[i] (may be NULL) the number of logits written. */
POCKET_TTS_API int pocket_tts_generate_ids(PocketTTSHandle handle, int n, const long long* const* ids, const int* n_ids,
                                           const float* const* voices, const int* voice_frames,
                                           const float* const* noise, AudioResult* results, float* const* latents_out,
                                           float* const* eos_out, int* frames_out, int* eos_count_out);

/* The same through the slot table (queue with slot refill, any n): utterances finish and are replaced independently. */
POCKET_TTS_API int pocket_tts_generate_ids_queued(PocketTTSHandle handle, int n, const long long* const* ids, const int* n_ids,
                                                  const float* const* voices, const int* voice_frames,
                                                  const float* const* noise, AudioResult* results, float* const* latents_out,
                                                  float* const* eos_out, int* frames_out, int* eos_count_out);

/* pocket_tts_generate_ids in three parts, for callers that time or overlap the device-resident middle:
 *   stage : host -> HBM copy of ids, conditioning rows and start points; returns a batch owned by the engine
 *           (valid until the next stage / generate call with the same n on this handle), or NULL;
 *   run   : prefill + frame loop + chunked decode; audio stays in HBM; frames_out[i] = frames of utterance i;
 *   fetch : HBM -> host; fills results[i] (release with pocket_tts_free_audio) and, if given, latents_out[i]. */
POCKET_TTS_API void* pocket_tts_stage_ids(PocketTTSHandle handle, int n, const long long* const* ids, const int* n_ids,
                                          const float* const* voices, const int* voice_frames, const float* const* noise);
POCKET_TTS_API int pocket_tts_run_staged(PocketTTSHandle handle, void* staged, int* frames_out);
POCKET_TTS_API int pocket_tts_fetch_staged(PocketTTSHandle handle, void* staged, const int* frames, AudioResult* results,
                                           float* const* latents_out);

/* Streaming from token ids; same schedule and callback contract as pocket_tts_generate_streaming.
 * Returns total samples or -1. */
POCKET_TTS_API int pocket_tts_streaming_ids(PocketTTSHandle handle, const long long* ids, int n_ids, const float* voice,
                                            int voice_frames, const float* noise, int chunk_size_frames,
                                            AudioChunkCallbackC callback, void* user_data);

/* Text pre-step alone: normalisation + SentencePiece ids (src/tokenizer.cpp:27-60).
 * Returns the id count (may exceed cap; only cap ids are written) or -1. */
POCKET_TTS_API int pocket_tts_tokenize(PocketTTSHandle handle, const char* text, long long* ids, int cap);

/* ---- one entry point per reference graph call ------------------------------------------------- */

/* text_conditioner: ids[T] -> out[T][d_model]                       (src/pocket_tts.cpp:299-320) */
POCKET_TTS_API int ptts_text_conditioner(PocketTTSHandle handle, const long long* ids, int T, float* out);

/* Recurrent state of `batch` lock-step utterances (LM KV caches + decoder state), zero-initialised
 * like the reference's initState (src/pocket_tts.cpp:133-186). */
POCKET_TTS_API void* ptts_state_new(PocketTTSHandle handle, int batch);
POCKET_TTS_API void ptts_state_free(PocketTTSHandle handle, void* state);
POCKET_TTS_API int ptts_state_reset(PocketTTSHandle handle, void* state);

/* The same with the LM's keys and values in a pool of `pages` pages of page_size rows that the slots share, up to max_context rows
 * each (ptts_paged_plan, ptts_rotary_append and ptts_paged_attention below run inside).  window > 0: a row sees the last `window` rows
 * and the first `sinks` ones, and pages behind the window return to the pool.  ptts_lm_prefill may be called repeatedly (a prompt
 * in chunks); a call that needs more pages than are free fails and changes nothing.  No counterpart in the reference. */
POCKET_TTS_API void* ptts_state_new_paged(PocketTTSHandle handle, int batch, int pages, int page_size, int max_context, int window, int sinks);
/* Slot to_slot of a paged state begins anew with the first `rows` rows of from_slot (one voice for many utterances): whole pages
 * are shared, the rest is copied.  The slot's own pages go back to the pool (and serve for the copy); rows that from_slot has given back
 * cannot be shared.  The LM's state alone: the codec's state of to_slot stays as it is. */
POCKET_TTS_API int ptts_state_share(PocketTTSHandle handle, void* state, int from_slot, int to_slot, int rows);
/* Free pages of a paged state's pool. */
POCKET_TTS_API int ptts_state_free_pages(PocketTTSHandle handle, void* state);

/* flow_lm_main, prefill shape: sequence empty, text_embeddings = emb[rows][d_model] for one utterance
 * (src/pocket_tts.cpp:572,575). */
POCKET_TTS_API int ptts_lm_prefill(PocketTTSHandle handle, void* state, int slot, const float* emb, int rows);

/* flow_lm_main, decode shape: sequence[batch][latent_dim] (NaN row = BOS), empty text
 * -> cond[batch][d_model], eos[batch]                               (src/pocket_tts.cpp:591-593). */
POCKET_TTS_API int ptts_lm_step(PocketTTSHandle handle, void* state, const float* sequence, float* cond, float* eos);

/* flow_lm_flow iterated lsd_steps times with the Euler update, fused on the GPU:
 * cond[rows][d_model], x0[rows][latent_dim] -> x[rows][latent_dim]  (src/pocket_tts.cpp:414-451, 615-622). */
POCKET_TTS_API int ptts_flow_euler(PocketTTSHandle handle, const float* cond, const float* x0, int rows, float* x);

/* ptts_flow_euler for callers that cannot allocate device memory (code under HIP graph capture, serving loops and
 * harnesses that forbid hipMalloc).  No counterpart in the reference.  cond, x0 and x are DEVICE pointers on the
 * handle's GPU (x must not alias x0); the scratch the kernels need (adaLN vectors, partial-sum slabs) is a static
 * device array of ptts_flow_euler_noalloc_capacity() bytes (32 MiB) that each GPU holds until the process ends.  The
 * call allocates and frees nothing, returns when x is complete, and fails with a message that names the limit when
 * `rows` needs more scratch than the array holds (full-size model at lsd_steps 10: 59 rows fit).  Calls on one GPU
 * share that GPU's array: the library serialises its own calls per GPU; do not run two processes' worth of
 * overlapping calls through other means. */
POCKET_TTS_API int ptts_flow_euler_noalloc(PocketTTSHandle handle, const float* cond_dev, const float* x0_dev, int rows, float* x_dev);
POCKET_TTS_API unsigned long long ptts_flow_euler_noalloc_capacity(void);

/* mimi_decoder on one chunk: latents[batch][n][latent_dim], n <= 15 -> audio[batch][n*samples_per_frame]
 * with the state carried in `state`                                 (src/pocket_tts.cpp:463-543). */
POCKET_TTS_API int ptts_mimi_decode(PocketTTSHandle handle, void* state, const float* latents, int n, float* audio);

/* mimi_encoder: audio[samples] at 24 kHz -> out[frames][d_model]; returns the frames the clip gives, or -1.  At most
 * cap_frames rows are written: a return value above cap_frames (>= 0) means the output was cut there
 *                                                                   (src/pocket_tts.cpp:261-291). */
POCKET_TTS_API int ptts_mimi_encode(PocketTTSHandle handle, const float* audio, int samples, float* out, int cap_frames);
/* The same over n_clips clips of `samples` samples each, stacked through the encoder together (the reference encodes one
 * clip per call, src/pocket_tts.cpp:241-297): outs[i] receives clip i's rows; returns the rows per clip (each outs[i] gets at
 * most cap_frames of them, as above). */
POCKET_TTS_API int ptts_mimi_encode_batch(PocketTTSHandle handle, const float* const* clips, int n_clips, int samples, float* const* outs,
                                          int cap_frames);

/* ---- keys and values in pages: plan, rotary append, attention ------------------------------------------------------------
 *
 * For serving loops that schedule by themselves: requests share a pool of pages instead of holding a slot of fixed length each
 * (ptts_state_new), so one voice's rows serve many utterances, prompts arrive in chunks and long streams keep a window.
 * One step of a model calls ptts_paged_plan once, then ptts_rotary_append and ptts_paged_attention for every layer.
 *
 * Unlike the calls above, these take DEVICE pointers of GPU `device`, enqueue on `stream` (a hipStream_t; NULL: the device's
 * default stream) and return without waiting: 0, or -1 with a message and nothing launched.  They allocate nothing, keep nothing
 * between calls, may be called from several threads at once and may be captured into a graph.  Buffers must not overlap unless
 * stated.  Addresses are multiples of their type's size.  Strides count elements; the last axis is contiguous.  Values in device memory (lengths, page ids, slots) are checked
 * by the kernels: what is out of range is not read or written and sets a bit of *status (may be NULL; the caller clears it):
 * 1 page id or slot outside the pool, 2 row ranges outside the rows or not ascending, 4 a length negative or beyond its table. */
enum { PTTS_TYPE_F32 = 0, PTTS_TYPE_BF16 = 1, PTTS_TYPE_F16 = 2 };

/* A pool of pages: key row r of page p and head h at k + p * page_stride + r * row_stride + h * head_stride, values likewise at v.
 * Pointers and strides are multiples of 16 bytes, head_dim is a multiple of 8 up to 256; any page_size, pages * page_size < 2^30. */
typedef struct {
    void* k;
    void* v;
    long long page_stride, row_stride, head_stride;
    int type, pages, page_size, kv_heads, head_dim;
} PttsPages;

/* Block tables and slot maps from request lengths, in one launch.  Request i holds cached[i] rows in the first
 * ceil(cached[i] / page_size) pages of its block_table row and receives arriving[i] more.  The pages it lacks are taken from
 * free_pages in order (request 0's first) and entered in its table row; other entries stay as they are.  Row r of the packed new
 * rows (request 0's first) gets positions[r] and slot_map[r] = page * page_size + row inside the page.  cu_rows[i] is the first
 * packed row of request i (requests + 1 entries), kv_len[i] = cached[i] + arriving[i].
 * counts[4] = new rows in all (those beyond `rows` are not written), pages taken, pages missing, rows without a page.  A page that is missing (free list exhausted, or
 * table row full) leaves -1 in the table and its rows get slot -1, in later plans too.  An id below 0 in free_pages is entered as it
 * is and its rows get slot -1 (status 1; counts takes it for a page).  A negative length counts as 0.
 * Rows of slot_map and positions behind the last new row stay as they are: a loop that gives ptts_rotary_append more rows than arrive
 * (a captured step of fixed size) sets its slot_map to -1 before the plan, or they name the slots of an earlier step.  The last page of a request must not be shared when
 * it is partly filled and rows arrive.  requests <= 65536. */
typedef struct {
    const int* cached;
    const int* arriving;
    const int* free_pages;
    int* block_table;
    int* slot_map;
    int* positions;
    int* cu_rows;
    int* kv_len;
    int* counts;
    int* status;
    long long table_stride;
    int requests, table_width, n_free, page_size, rows;
} PttsPagedPlan;
POCKET_TTS_API int ptts_paged_plan(const PttsPagedPlan* plan, int device, void* stream);

/* Rotary frequencies for ptts_rotary_append, on the host: out[rot_dim / 2] in radians per position; *magnitude (may be NULL) is the
 * factor for the rotated values.  scaling 0: base^(-2 i / rot_dim).  1: positions divided by `factor`.  2: the base stretched so
 * that the lowest frequency is divided by `factor` and the highest kept.  3: by parts: frequencies that turn more than `fast`
 * times within `trained` positions are kept, those below `slow` turns are divided by `factor`, a linear ramp in between, and
 * magnitude = 0.1 ln(factor) + 1. */
POCKET_TTS_API int ptts_rotary_frequencies(int rot_dim, double base, int scaling, double factor, double trained, double fast, double slow,
                                           double* out, float* magnitude);

/* Rotates the first rot_dim values of every head of q and k by positions[row] * freq[i] (device, float64: far positions keep their
 * angle), pairs (2 i, 2 i + 1) if interleaved, else (i, i + rot_dim / 2), times `magnitude`; the rest of the head passes unscaled.  q goes to q_out (q itself
 * is allowed, with the same strides).  k and v go to the pages, row r to slot slot_map[r] (-1: not stored).  Two rows must not
 * name one slot; rows < 2^24.  q, or k and v (then pages and slot_map too), may be NULL.  q, q_out, k and v have `type`; the pages
 * have the same, or bf16 under f32 rows (rounded to nearest even). */
typedef struct {
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    const int* positions;
    const int* slot_map;
    const double* freq;
    int* status;
    long long q_row_stride, q_head_stride, k_row_stride, k_head_stride, v_row_stride, v_head_stride, out_row_stride, out_head_stride;
    PttsPages pages;   /* without k and v only head_dim is read */
    float magnitude;
    int type, rows, q_heads, rot_dim, interleaved;
} PttsRotaryAppend;
POCKET_TTS_API int ptts_rotary_append(const PttsRotaryAppend* args, int device, void* stream);

/* Attention of every request's new rows over its pages.  Rows cu_rows[i] .. cu_rows[i + 1] - 1 of q are request i's last positions,
 * kv_len[i] - 1 for the last of them (so their own keys are in the pages already).  The query at position p sees key j if j <= p and
 * (window <= 0 or j > p - window or j < sinks).  out = softmax(scale q.k) v, lse (may be NULL) = ln sum exp(scale q.k); a row that
 * sees nothing gets 0 and -inf.  Head h of q reads head h / (q_heads / kv_heads) of the pages.  Keys that a row does not see
 * never reach it, whatever they hold.  A key that a row sees and whose page id is not one of the pool's (-1 of a plan that ran out of
 * pages too) counts as a row of zeros, in k and in v, and sets status 1: check the plan's counts or the status.  out may not alias q.
 * rows * (q_heads / kv_heads) < 2^30.  Types: q and out q_type; pages of q_type, or bf16 pages under f32 rows.  q and out and their strides
 * are multiples of 16 bytes.  Rows outside every request stay as they were.
 * Rounding: scores, softmax statistics and sums are float32; bf16 and f16 rows round each weight to their type before it meets its value
 * (half a step on each weight, beside the result's own half step), f32 rows keep float32 weights.
 * max_rows, max_kv: what the caller knows of the largest row count and length of a request (0: nothing).  They choose how the work
 * is cut and cost time when wrong, never results.
 * workspace: ptts_paged_attention_workspace() bytes (0: none needed; -1: bad arguments), 16-byte aligned, contents irrelevant
 * before and after; concurrent calls (and graphs that may run at the same time) need one each. */
typedef struct {
    const void* q;
    void* out;
    float* lse;
    const int* cu_rows;
    const int* kv_len;
    const int* block_table;
    int* status;
    void* workspace;
    long long q_row_stride, q_head_stride, out_row_stride, out_head_stride, lse_row_stride, table_stride, workspace_bytes;
    PttsPages pages;
    float scale;
    int q_type, rows, requests, q_heads, table_width, window, sinks, max_rows, max_kv;
} PttsPagedAttention;
POCKET_TTS_API long long ptts_paged_attention_workspace(const PttsPagedAttention* args, int device);
POCKET_TTS_API int ptts_paged_attention(const PttsPagedAttention* args, int device, void* stream);

/* ---- host-side pre/post steps, usable without a GPU ---------------------------------------------- */

/* Text pre-step on its own (src/tokenizer.cpp:14-60).  raw != 0 skips the sentence clean-up. */
POCKET_TTS_API void* ptts_tokenizer_new(const char* model_path);
POCKET_TTS_API void ptts_tokenizer_free(void* tokenizer);
POCKET_TTS_API int ptts_tokenizer_vocab(void* tokenizer);
POCKET_TTS_API int ptts_tokenizer_encode(void* tokenizer, const char* text, int raw, long long* ids, int cap);

/* AudioUtils of the reference (src/audio_utils.cpp:45-303).  Each returns the output length (writing at
 * most cap samples) or -1. */
POCKET_TTS_API int ptts_audio_load_wav(const char* path, int target_rate, float* out, int cap);
POCKET_TTS_API int ptts_audio_save_wav(const char* path, const float* samples, int n, int rate);
POCKET_TTS_API int ptts_audio_resample(const float* in, int n, int in_rate, int out_rate, float* out, int cap);
POCKET_TTS_API int ptts_audio_normalize(const float* in, int n, float* out);

/* Benchmark support: HIP-event timing on the streams the engine launches on.  Both arrays hold 4 entries:
 * [0] LM frame step (kernel chain), [1] flow phase (adaLN GEMMs + fused head), [2] decoder chunk,
 * [3] the flow head's launch chain alone (lsd_steps * (blocks + 1) launches per frame, counted in calls[3]);
 * times_ms = totals, calls = number of launches of each. */
/* The int8 matrix product of the "int8" precision on its own: out[M][N] = A[M][K] . W[N][K]^T with W quantised per
 * output row to int8 and A per row and per block of 64 k (K % 64 == 0, N % 16 == 0).  For checking the kernel's
 * arithmetic exactly; the model paths call the same kernel. */
POCKET_TTS_API int ptts_q8_linear(PocketTTSHandle handle, const float* A, int M, int K, const float* W, int N, float* out);
/* The same with the matrix given in int8 form, q[N][K] and one scale per output row (what a pack's `<name>.q8` carries). */
POCKET_TTS_API int ptts_q8_linear_q(PocketTTSHandle handle, const float* A, int M, int K, const signed char* q, const float* scale, int N,
                                    float* out);

/* The same product in the int8 engine's second activation scheme, the one ONNX Runtime's dynamically quantised graphs
 * use (DynamicQuantizeLinear + MatMulInteger; the reference's *_int8.onnx models, src/pocket_tts.cpp:232-246): each row
 * of A becomes uint8 with one scale and one zero point over the whole row (range widened to include 0), W is int8 per
 * output row, the integer sum runs over all of K and is scaled once. */
POCKET_TTS_API int ptts_q8_linear_dyn(PocketTTSHandle handle, const float* A, int M, int K, const float* W, int N, float* out);

/* The bf16-weight matrix product on its own: out[M][N] = act(A . W^T + bias) * colscale + R (bias, colscale, R may be
 * NULL; act: 0 none, 1 GELU, 2 SiLU, 3 ELU; W is rounded to bf16).  flags bit 0: carry A as two bf16 terms; bit 1: keep
 * the A rows in bf16 in device memory; bit 2: keep the C rows in bf16.  For checking the kernels at arbitrary shapes; the
 * model paths go through the same dispatch. */
POCKET_TTS_API int ptts_bf16_linear(PocketTTSHandle handle, const float* A, int M, int K, const float* W, int N, const float* bias,
                                    const float* colscale, const float* R, int act, int flags, float* out);

POCKET_TTS_API int ptts_phase_timing(PocketTTSHandle handle, int enable);
/* The slot table that serves pocket_tts_generate, pocket_tts_generate_streaming, pocket_tts_generate_batch and the _queued calls:
 * stats[0] = activations of the table (idle -> busy), stats[1] = utterances served, stats[2] = most slots occupied at once. */
POCKET_TTS_API int ptts_scheduler_stats(PocketTTSHandle handle, long* stats);
/* ... and stats[3] = frame steps launched, [4] = sum of the launch width over them, [5] = frames delivered to callers,
 * [6] = decoder chunk calls, [7] = prefill passes (8 entries). */
POCKET_TTS_API int ptts_scheduler_stats_ex(PocketTTSHandle handle, long* stats);
/* Engines behind the handle: one per GPU listed in the environment variable POCKET_TTS_DEVICES (e.g. "0,1,2,3") when the
 * handle was created, else one.  served[i] (i < cap, may be NULL) receives the utterances engine i has served.  Single
 * utterances and streams go to the engine with the fewest utterances pending, queued batches are dealt out over all. */
POCKET_TTS_API int ptts_engine_count(PocketTTSHandle handle, long* served, int cap);
POCKET_TTS_API int ptts_phase_times(PocketTTSHandle handle, double* times_ms, long* calls);
/* bytes[0..3] = GEMM weight bytes (compute precision) of the LM, the flow head, the decoder, the encoder */
POCKET_TTS_API int ptts_weight_bytes(PocketTTSHandle handle, unsigned long long* bytes);

/* Weights carried by an ONNX file: graph initializers and Constant-node tensors, read at the protobuf wire level
 * (no onnx / protobuf dependency).  The reference gives its five .onnx graphs to ONNX Runtime
 * (src/pocket_tts.cpp:90-113); a converter (pocket-tts.cpp_amd/tools/onnx_to_ptts.py) uses these calls to build the
 * engine's weight pack from them.  dtype values are onnx.TensorProto.DataType (1 float, 2 uint8, 3 int8, 6 int32,
 * 7 int64, 10 float16, 11 double, 16 bfloat16).  read_f32 converts any of those to float; dequantize returns
 * (q - zero_point) * scale for the <base>_quantized / <base>_scale / <base>_zero_point triplets that ONNX Runtime's
 * quantisation tools write (axis -1: the one axis whose extent equals the number of scales).  Both return the
 * element count or -1.  Host only: usable without a GPU. */
POCKET_TTS_API void* ptts_onnx_open(const char* path);
POCKET_TTS_API void ptts_onnx_close(void* onnx);
POCKET_TTS_API int ptts_onnx_tensor_count(void* onnx);
POCKET_TTS_API int ptts_onnx_tensor_info(void* onnx, int index, const char** name, int* dtype, int* rank, long long* dims8);
POCKET_TTS_API int ptts_onnx_find(void* onnx, const char* name);
POCKET_TTS_API long long ptts_onnx_read_f32(void* onnx, int index, float* out, long long cap);
POCKET_TTS_API long long ptts_onnx_dequantize(void* onnx, const char* base, int axis, float* out, long long cap, int* rank, long long* dims8);
POCKET_TTS_API int ptts_onnx_node_count(void* onnx);
POCKET_TTS_API int ptts_onnx_node_info(void* onnx, int index, char* op_type, char* inputs, char* outputs, int cap);

#ifdef __cplusplus
}
#endif

#endif /* POCKET_TTS_AMD_H */
