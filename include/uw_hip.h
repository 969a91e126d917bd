/* C ABI of libuw_hip.so: the MI355X (gfx950) implementation of urro_whisper's transcription hot path.
 *
 * The reference (urroxyz/whisper, pure Python) reaches its numerics through four seams; each entry point
 * below replaces one of them and cites it.  A Python binding over ctypes is in whisper_amd/lib.py.
 *
 * Conventions: every function returns 0 on success, non-zero otherwise (uw_last_error() then holds a
 * message for the calling thread); nothing throws across the boundary.  Unless stated otherwise pointers are
 * DEVICE pointers owned by the caller, work is enqueued on `stream` (a hipStream_t passed as void*, NULL =
 * default stream) and is asynchronous.  A context belongs to one GPU and one caller thread at a time.
 */
#ifndef UW_HIP_H
#define UW_HIP_H
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

typedef struct uw_ctx uw_ctx;

#define UW_DTYPE_F32 0   /* exact-fp32 MFMA path: parity runs                     */
#define UW_DTYPE_BF16 1  /* bf16 operands, fp32 accumulate and residual stream    */
#define UW_MAX_ALIGN_HEADS 32

typedef struct uw_config {
    int32_t d_model, n_heads, enc_layers, dec_layers, vocab, n_mels;
    int32_t n_audio_ctx;   /* 1500 */
    int32_t n_text_ctx;    /* 448  */
    int32_t dtype;         /* UW_DTYPE_*                                            */
    int32_t max_batch;     /* windows in flight; sizes the workspace                */
    int32_t n_align_heads; /* alignment heads, (layer, head) pairs below            */
    int32_t align_layer[UW_MAX_ALIGN_HEADS];
    int32_t align_head[UW_MAX_ALIGN_HEADS];
} uw_config;

const char* uw_last_error(void);
int uw_abi_version(void);

/* Model loader seam: urro_whisper/model/load.py:13-98 builds two onnxruntime sessions from the encoder
 * and decoder graphs.  Here the graphs' initialisers arrive as `n_weights` fp32 device tensors in the
 * order of whisper_amd.weights.tensor_plan (HF WhisperForConditionalGeneration naming); the context keeps
 * its own packed copies (compute dtype, fused QKV, q pre-scaled by 1/8, conv kernels tap-major) plus the
 * whole workspace, so the caller may free the inputs afterwards.  `mel_filters` is a HOST pointer to the
 * [n_mels][201] fp32 Slaney filterbank.  Synchronous. */
int uw_ctx_create(const uw_config* cfg, const void* const* weights, int n_weights, const float* mel_filters,
                  uw_ctx** out);
int uw_ctx_destroy(uw_ctx* ctx);
/* bytes of device memory the context holds */
int64_t uw_ctx_bytes(const uw_ctx* ctx);

/* Decode steps (uw_decode_step, uw_decode_greedy, uw_transcribe_windows) read the cross-attention K/V from an 8-bit copy that
 * uw_cross_kv fills: format UW_KV8_INT8 or UW_KV8_E4M3, a scale per 64 frames and head (the paged cache below), or -1 for the compute
 * dtype again.  It halves the stream that bounds a step; multi-token passes keep reading the compute dtype.  Allocates on its
 * first use, synchronises, and asks for a new uw_cross_kv.  No counterpart in the reference. */
int uw_ctx_cross_cache(uw_ctx* ctx, int format);

/* Mel seam: calculate_mel_for_segment (urro_whisper/audio/load.py:67-121), i.e.
 * whisper.log_mel_spectrogram(audio, n_mels, padding=480000)[:, :3000].
 * audio: f32 [B][stride] 16 kHz PCM, n_samples: i32 [B] valid samples per window (<= stride),
 * mel_out: f32 [B][n_mels][3000]. */
int uw_mel(uw_ctx* ctx, const float* audio, int64_t stride, const int32_t* n_samples, int B, float* mel_out,
           void* stream);

/* Encoder seam: encoder_sess.run(None, {input_features: mel}) (urro_whisper/core.py:824-830).
 * mel: f32 [B][n_mels][3000] -> enc_out: f32 [B][1500][d_model] (may be NULL: result stays in the context). */
int uw_encode(uw_ctx* ctx, const float* mel, int B, float* enc_out, void* stream);

/* The reference re-projects the encoder states to cross-attention K/V inside every decoder run
 * (core.py:942-949); this does it once per window batch.  enc_states: f32 [B][1500][d_model], or NULL to use
 * the output of the last uw_encode. */
int uw_cross_kv(uw_ctx* ctx, const float* enc_states, int B, void* stream);

/* Decoder seam, cache-less form: decoder_sess.run(["logits"] | cross_attentions.*, {input_ids,
 * encoder_hidden_states}) (core.py:941-949, align.py:608-618).  Uses the K/V of the last uw_cross_kv.
 * ids: i32 [B][ld_ids], every window T tokens.  Optional outputs (NULL to skip):
 *   logits_all   f32 [B][T][vocab]
 *   logits_last  f32 [B][vocab]           (position T-1)
 *   cross_probs  f32 [dec_layers][B][n_heads][T][1500]   softmax probabilities. */
int uw_decoder_forward(uw_ctx* ctx, const int32_t* ids, int ld_ids, int B, int T, float* logits_all,
                       float* logits_last, float* cross_probs, void* stream);

/* Decoder seam, KV-cached form: one decoder_sess.run of the greedy loop (core.py:941-949) for the newest token
 * only.  The reference's decoder declares past_key_values.* inputs but always feeds them empty (core.py:185-192,
 * 943-946) and so re-runs the whole prefix; here the self-attention K/V of earlier positions stay in the context
 * (written by uw_decoder_forward or by earlier steps), so window b's positions 0..pos[b]-1 must have been
 * processed first.  ids, pos: i32 [B] device arrays; logits: f32 [B][vocab] for the token at pos[b].  A pos
 * outside 0..n_text_ctx-1 skips that window.  Invalidates the state of a uw_decode_greedy in progress. */
int uw_decode_step(uw_ctx* ctx, const int32_t* ids, const int32_t* pos, int B, float* logits, void* stream);

/* Greedy loop seam: core.py:938-968 plus the text filter of core.py:991, KV-cached.  prompt_ids: i32
 * [B][ld_prompt], prompt_len: i32 [B] HOST array, max_tokens: total sequence budget (prompt included).
 * Outputs (device): new_tokens i32 [B][n_text_ctx], n_new i32 [B], text_ids i32 [B][n_text_ctx], n_text i32 [B].
 * While decoding, the alignment heads' cross-attention rows are written into the context's rows buffer;
 * windows whose text continues after a generated non-text token get their rows from one teacher-forced
 * pass over prompt + text[:-1] (identical to the reference's per-token replay, align.py:603-630).
 * Synchronises the stream (the number of steps depends on the tokens). */
int uw_decode_greedy(uw_ctx* ctx, const int32_t* prompt_ids, int ld_prompt, const int32_t* prompt_len_host, int B,
                     int max_tokens, int eot, int sot, int ts_begin, int ts_end, int32_t* new_tokens, int32_t* n_new,
                     int32_t* text_ids, int32_t* n_text, void* stream);

/* Per-window outcome of the last uw_decode_greedy / uw_transcribe_windows on this context (both synchronise, so the
 * answer is complete when they return).  status: i32 [B] HOST array; 0 = decoded normally; 1 = the decoder produced a
 * logits row holding a NaN and the window stopped there, keeping the tokens generated before it -- the reference's
 * decoder-run failure inside the generation loop (core.py:948-956, 978-980: error stored, partial tokens kept). */
int uw_window_status(uw_ctx* ctx, int B, int32_t* status_host);

/* Alignment rows for a given text (forced alignment, align.py:446-471 / 603-630): one teacher-forced pass over
 * prompt + text[:-1]; rows land in the context's rows buffer.  All arrays device except the *_host lengths. */
int uw_attn_rows_forced(uw_ctx* ctx, const int32_t* prompt_ids, int ld_prompt, const int32_t* prompt_len_host,
                        const int32_t* text_ids, int ld_text, const int32_t* n_text_host, int B, void* stream);

/* Copies the context's rows buffer out: rows f32 [B][n_align_heads][n_rows][1500]. */
int uw_get_attn_rows(uw_ctx* ctx, int B, int n_rows, float* rows, void* stream);

/* perform_word_alignment's numeric front half (align.py:758-811,818): head mean, median filter 7 ('reflect'),
 * softmax, negate, f64.  rows f32 [B][n_sel][n_rows_max][S]; n_tok i32 [B] (device); cost f64 [B][n_rows_max][S]. */
int uw_cost_matrix(const float* rows, int n_sel, const int32_t* n_tok, int B, int n_rows_max, int S, double* cost,
                   void* stream);

/* dtw.dtw(cost, step_pattern=symmetric1) + boundary extraction (align.py:818-853).  cost f64 [B][n_rows_max][S];
 * n_tok i32 [B]; dir_ws: scratch of uw_dtw_workspace_bytes(); boundaries i32 [B][n_rows_max+1] (n_tok[b]+1 used);
 * optional path_i/path_j i32 [B][n_rows_max+S] and path_len i32 [B].
 * A window without a warping path (a NaN or infinite cost leaves cells without a predecessor; the reference returns
 * no timestamps when dtw raises, align.py:823-827) gets boundaries[b][0] = -1 and path_len[b] < 0; the call itself
 * still returns 0 because the other windows of the batch are valid. */
int64_t uw_dtw_workspace_bytes(int B, int n_rows_max, int S);
int uw_dtw(const double* cost, const int32_t* n_tok, int B, int n_rows_max, int S, void* dir_ws, int32_t* boundaries,
           int32_t* path_i, int32_t* path_j, int32_t* path_len, void* stream);

/* uw_dtw for callers that cannot allocate or hand over a workspace (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc).  No counterpart in the reference.  Same inputs, outputs and results as
 * uw_dtw; the direction matrix lives in a fixed 16 MiB device array inside the library (one per GPU, held until the
 * process ends), so B * n_rows_max * ceil(S / 16) * 4 bytes must not exceed 16 MiB (e.g. 95 windows x 448 rows x 1500
 * frames) -- larger problems are rejected with an error, use uw_dtw.  The call allocates nothing.  All calls on one GPU
 * share the array: calls that overlap on one GPU (different streams or threads) race.  The array of the CURRENT device is
 * used, so the device that owns `cost`, the outputs and `stream` must be current when the call is made (a cost matrix on
 * another device is rejected). */
#define UW_DTW_STATIC_BYTES (16 << 20)
int uw_dtw_static(const double* cost, const int32_t* n_tok, int B, int n_rows_max, int S, int32_t* boundaries,
                  int32_t* path_i, int32_t* path_j, int32_t* path_len, void* stream);

/* cost matrix + DTW on the context's rows buffer: boundaries i32 [B][n_text_ctx+1]. n_text i32 [B] device.
 * boundaries[b][0] = -1 marks a window for which no path exists (see uw_dtw). */
int uw_align(uw_ctx* ctx, const int32_t* n_text, int B, int32_t* boundaries, void* stream);

/* The whole path for a batch of windows: mel -> encoder -> cross K/V -> greedy decode with row capture ->
 * cost matrix -> DTW (core.py:798-1030 numerics).  Same outputs as uw_decode_greedy plus boundaries.
 * A context created without alignment heads (the reference's "no alignment" case, align.py:81-84,595-597) skips the
 * cost matrix and DTW and fills boundaries with -1; boundaries[b][0] = -1 always means "window b has no timestamps". */
int uw_transcribe_windows(uw_ctx* ctx, const float* audio, int64_t stride, const int32_t* n_samples,
                          const int32_t* prompt_ids, int ld_prompt, const int32_t* prompt_len_host, int B, int max_tokens,
                          int eot, int sot, int ts_begin, int ts_end, int32_t* new_tokens, int32_t* n_new,
                          int32_t* text_ids, int32_t* n_text, int32_t* boundaries, void* stream);

/* Measurement aid (no reference counterpart): brackets every launch of the cross-attention decode kernel --
 * the kernel that streams the cross K/V cache and bounds the path -- with HIP events on the caller's stream.
 * uw_profile_end synchronises the device and returns how many launches ran, how many were timed (the event
 * pool holds max_launches pairs), how many windows those launches covered in total (a launch streams the K/V
 * of one decoder layer for its windows) and the summed duration of the timed ones. */
int uw_profile_begin(uw_ctx* ctx, int max_launches);
int uw_profile_end(uw_ctx* ctx, int64_t* launches_total, int64_t* launches_timed, int64_t* windows_total,
                   double* timed_ms);
/* Between the same begin / end, four more spans are bracketed with events, sparsely: kind 1 = launches of the
 * self-attention decode kernel (one in eight timed), 2 = the encoder pass of uw_transcribe_windows, 3 = the DTW launch
 * of uw_align, 4 = whole decode steps of the greedy loop (all launches of one step; one step in eight timed).  Read after
 * uw_profile_end: how many ran, how many were timed, the summed duration of the timed ones. */
int uw_profile_span(uw_ctx* ctx, int kind, int64_t* launches_total, int64_t* launches_timed, double* timed_ms);

/* ---- 8-bit paged key/value cache and draft verification -------------------------------------------------------------
 * Context-free operators for serving (no counterpart in the reference, which feeds its past_key_values.* empty,
 * core.py:185-192).  They work on the CURRENT device, allocate nothing, never synchronise and may be captured into a graph.
 *
 * The cache is four arrays the caller owns.  A page ("block") holds `page` tokens of all kv heads:
 *   k        8-bit codes [n_pages][n_kv_heads][page][head_dim]
 *   v        8-bit codes [n_pages][n_kv_heads][head_dim][page]   (transposed inside the page)
 *   k_scale, v_scale  f32 [n_pages][n_kv_heads];   value = code * scale
 * Formats: UW_KV8_INT8 (codes -127..127) and UW_KV8_E4M3 (1-4-3 without infinities, scales are powers of two).  page: 16, 32,
 * 64, 128 or 256; head_dim: 64 or 128.  k and v must be 16-byte aligned.
 * (What a cache that was filled otherwise has to keep: codes of tokens are numbers, scales 0 -- all codes of the block 0 -- or 2^-126 at
 * least, or NaN.  Codes behind a sequence's end may be anything.)
 * table i32 [B][table_width]: the page of each block of a sequence, block i holding positions i * page ... Entries behind a
 * sequence's end are not read.  A page id outside 0..n_pages-1, or a position before 0 or behind the table, is never accessed:
 * an append skips it, a read and an attention row that sees it give NaN.
 * Tokens come either T per sequence (tok_start NULL, T > 0, n_tok = B * T), sequence b's first row at b * seq_stride, or packed
 * one sequence behind the other (tok_start i32 [B+1], row r at r * tok_stride; T and seq_stride are ignored); rows behind
 * tok_start[B] are neither read nor written.  Strides are in elements; element (row, head, i) lies at row + head * head_stride + i;
 * base pointers and strides must be multiples of 16 bytes.  dtype: UW_DTYPE_F32 or UW_DTYPE_BF16. */
#define UW_KV8_INT8 0
#define UW_KV8_E4M3 1
typedef struct uw_kv8_cache {
    void *k, *v;
    float *k_scale, *v_scale;
    int32_t n_pages, n_kv_heads, page, head_dim, format, reserved;
} uw_kv8_cache;
typedef struct uw_kv8_seqs {        /* the sequences of a call and how the rows of its token arrays belong to them */
    const int32_t *table, *len;     /* page table; [B] positions or lengths, see the calls */
    const int32_t* tok_start;
    int64_t n_tok;
    int32_t table_width, B, T, dtype;
} uw_kv8_seqs;
typedef struct uw_kv8_tokens {      /* a [rows][heads][head_dim] array */
    void* data;
    int64_t seq_stride, tok_stride, head_stride;
} uw_kv8_tokens;
typedef struct uw_kv8_store_args {
    uw_kv8_cache cache;
    uw_kv8_seqs seqs;
    uw_kv8_tokens k, v;
} uw_kv8_store_args;
typedef struct uw_kv8_attention_args {
    uw_kv8_cache cache;
    uw_kv8_seqs seqs;
    uw_kv8_tokens q, o;
    float* lse;
    void* ws;
    int64_t ws_bytes;
    int32_t n_heads, causal;
    float scale;
    int32_t reserved;
} uw_kv8_attention_args;

/* Appends keys and values: sequence b's tokens go to positions len[b], len[b] + 1, ... (len = tokens already there).
 * Per touched block, head and half: a block without earlier tokens takes its scale from the largest |x| (int8: |x| times the f32
 * next to 1/127, 2^-126 at least; e4m3: the smallest power of two that leaves codes up to 448); otherwise the scale
 * stays while the new values fit and grows by a power of two if not, the earlier tokens' codes being re-rounded.  A NaN or
 * infinity makes the scale of its block and head NaN until the block is begun again: whatever reads that block gives NaN.
 * A page must not be touched twice by one call, from two sequences or two blocks of one (shared prefixes end on a page boundary).  Codes behind the last
 * token are left as they are. */
int uw_kv8_append(const uw_kv8_store_args* args, void* stream);
/* Reads tokens back as values (code * scale in f32, that rounded to dtype): positions len[b], len[b] + 1, ... into k and v. */
int uw_kv8_read(const uw_kv8_store_args* args, void* stream);
/* Attention of n_heads query heads (a multiple of n_kv_heads; query head h reads kv head h / (n_heads / n_kv_heads)) over the
 * first len[b] cached tokens; with causal != 0 token t of the n tokens of a sequence sees keys 0 .. len[b] - n + t (its own
 * key, appended before, is the last).  o: rows like q; lse (may be NULL) f32 [n_tok][n_heads]: log of the sum of exp(scores).
 * A row that sees no key (len[b] <= 0 among others) gives 0 and lse = -inf.  scale (finite) multiplies q.k.  ws: ws_bytes of scratch, at least what
 * uw_kv8_attention_workspace_bytes() answers for the same arguments (it reads no device memory; -1: arguments refused),
 * 16-byte aligned, not shared by calls that may run at the same time; NULL if that is 0. */
int64_t uw_kv8_attention_workspace_bytes(const uw_kv8_attention_args* args);
int uw_kv8_attention(const uw_kv8_attention_args* args, void* stream);

/* Verification of drafted tokens (speculative decoding): target [B][N+1][V] and draft [B][N][V] (NULL: the drafter is taken to
 * have been certain of its token) are logits, or probabilities if `probs`; rows at b * *_sB + i * *_sN, elements contiguous.
 * drafted i32 [B][N], n_drafted i32 [B] (NULL: N for all; clamped to 0..N), uniforms f32 [B][N+1] in [0, 1).
 * With p_i, q_i = softmax(row / temperature): token i is accepted while uniforms[b][i] * q_i(d_i) < p_i(d_i).  At the first
 * rejection the next token is drawn from max(p_i - q_i, 0), after the last accepted one from p_n: the smallest index whose
 * cumulative weight exceeds uniforms[b][N] times the whole.  All of this in 64-bit numbers, the temperature too; an exponential is off by
 * 1.1e-12 at most.  temperature 0: a token is accepted while it
 * is its row's arg-max (the lowest index of equal ones) and the next token is the arg-max; draft and uniforms are not read.
 * accepted i32 [B]; tokens i32 [B][N+1]: the accepted tokens, the next token, then -1.  The next token is -1 if its row holds
 * a NaN or has no mass -- at temperature 0 a NaN only -- (the decoder-run failure of core.py:948-956); a drafted id outside 0..V-1 is never accepted.
 * ws: ws_bytes of scratch, at least uw_verify_draft_workspace_bytes() (-1: arguments refused), 16-byte aligned, not shared by
 * calls that may run at the same time. */
typedef struct uw_verify_args {
    const void* target;
    int64_t target_sB, target_sN;
    const void* draft;
    int64_t draft_sB, draft_sN;
    const int32_t *drafted, *n_drafted;
    const float* uniforms;
    int32_t *accepted, *tokens;
    void* ws;
    int64_t ws_bytes;
    int32_t dtype, B, N, V;
    double temperature;
    int32_t probs, reserved;
} uw_verify_args;
int64_t uw_verify_draft_workspace_bytes(const uw_verify_args* args);
int uw_verify_draft(const uw_verify_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif
