/* C ABI of the MI355X decode engine (libillhip.so).
 *
 * Drop-in for the pass API of the reference's Swift `Engine`
 * (Sources/Engine/Engine.swift); the reference's only C ABI is the one-function shim
 * Sources/CShim/include/cshim.h:3-4, which this header extends in the same style: plain
 * C types, an opaque handle, no GPU types in the signatures.
 *
 * Conventions: every function returns 0 on success or a negative error code; the message
 * of the last error on the calling thread is available from ill_last_error(). The caller
 * owns host arrays; the engine owns device memory. An engine is single-threaded and runs
 * on one HIP stream of one GPU.
 */
#ifndef ILL_HIP_H
#define ILL_HIP_H
#include <stdint.h>

/* The library is built with hidden visibility: these entry points are its only exports. */
#ifndef ILL_API
#define ILL_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ill_engine ill_engine;

enum {
  ILL_OK = 0,
  ILL_E_ARG = -1,      /* bad argument (shape, size, state) */
  ILL_E_FILE = -2,     /* model file missing or malformed */
  ILL_E_HIP = -3,      /* HIP runtime error */
  ILL_E_TIMEOUT = -4,  /* a device-side bounded wait expired (the pass was abandoned) */
  ILL_E_FORMAT = -5    /* weight format not supported by this build */
};

/* Thread-local message of the last failure (never NULL). */
ILL_API const char* ill_last_error(void);

/* Engine(modelPath:maxContext:maxPass:maxSteps:) (Engine.swift:71-232): maps the .ill v1
 * file (ModelFile.swift:73-98), repacks the weights into the device tile layout and copies
 * them to HBM once. max_context is rounded up to a multiple of 64. */
ILL_API int ill_create(const char* ill_path, int max_context, int max_pass, int max_steps, ill_engine** out);
ILL_API int ill_destroy(ill_engine* e);

/* Model facts of the loaded file. */
ILL_API int ill_vocab(const ill_engine* e);
ILL_API int ill_layers(const ill_engine* e);
ILL_API int ill_format(const ill_engine* e);   /* 0 f16, 1 q8, 2 q4 */

/* The 16-int device State (Shaders.swift:37-54): pos, n, step, done, maxctx, maxsteps,
 * eos0, eos1, nver, tspec, passes, accepted, tlmh, nodraft, learned, tree.
 * Host writes it before a request (Engine.swift:945-964). */
ILL_API int ill_set_state(ill_engine* e, const int32_t state[16]);
ILL_API int ill_get_state(ill_engine* e, int32_t state[16]);

/* encodePrefill (Engine.swift:588-601): n tokens at positions state.pos.., lm_head on the
 * last row and a greedy commit (the first generated token lands in out_tokens[step] and
 * becomes the next step's input). write_logits keeps that row's fp32 logits. */
ILL_API int ill_prefill(ill_engine* e, const int32_t* toks, int n, int write_logits);

/* encodeDecodeStep (Engine.swift:605-609): one 1-row step on the last committed token. */
ILL_API int ill_decode_step(ill_engine* e, int write_logits);

/* encodeWidePass / encodeSpecPass + k_commit_spec (Engine.swift:567-579, :503-547;
 * Shaders.swift:246-418 without drafting): one pass over `rows` (<= 16) rows.
 * tree != NULL: the 65-int tree [n, depth[16], parent[16], tok[16], anc[16]] with tok[0] =
 * the last committed token; rows attend to the context and their ancestors, the longest
 * path whose drafts equal their parent's argmax is committed and its K/V compacted.
 * tree == NULL: a chain of toks[0..rows-1] = [last token, drafts...]. */
ILL_API int ill_verify_pass(ill_engine* e, int rows, const int32_t* tree, const int32_t* toks, int write_logits);

/* Record `nsteps` decode steps into one hipGraph; ill_launch_graph replays it. Steps after
 * the stop flag early-exit on the device (Shaders.swift:41). The device also sets the stop
 * flag once a following pass of up to 16 rows would not fit in the context, and
 * ill_set_state refuses a live state without that room, so replays never write K/V past
 * max_context. A captured graph is dropped when tracing is switched on or off. */
ILL_API int ill_capture_steps(ill_engine* e, int nsteps);
ILL_API int ill_launch_graph(ill_engine* e);
/* ill_launch_graph with encodeDecodeStep's writeLogits (Engine.swift:605-609) for every
 * recorded step: afterwards ill_read_logits(e, 0, ..) holds the last executed step's logits. */
ILL_API int ill_launch_graph_logits(ill_engine* e, int write_logits);

ILL_API int ill_sync(ill_engine* e);

/* Pinned host array [max_steps] of committed tokens (-1 = not yet written): poll it with
 * volatile loads, as the reference does with ill_volatile_load (cshim.h:4). */
ILL_API const int32_t* ill_out_tokens(ill_engine* e);
ILL_API int ill_reset_out_tokens(ill_engine* e);

/* fp32 logits of pass row `row` from the last pass that wrote logits ([vocab] floats). */
ILL_API int ill_read_logits(ill_engine* e, int row, float* out);

/* Prefix K/V save/load (Engine.swift:788-838) in the reference cache layout:
 * [layer][kv_head][npos][64] f16 bits, for positions 0..npos-1. */
ILL_API int ill_kv_copy_out(ill_engine* e, int npos, uint16_t* k, uint16_t* v);
ILL_API int ill_kv_copy_in(ill_engine* e, int npos, const uint16_t* k, const uint16_t* v);

/* Engine.generate (Engine.swift:922-1038) for one request without drafting: sets the
 * state, prefills `ntok` tokens, then runs decode steps in captured graphs of `chunk`
 * steps while polling out_tokens. Writes up to max_new tokens (stop token excluded) to
 * out and returns their count through n_out; logits_out (optional, [vocab]) receives the
 * first token's logits. */
ILL_API int ill_generate(ill_engine* e, const int32_t* toks, int ntok, int max_new, int chunk,
                 int32_t* out, int* n_out, float* logits_out);

/* Engine.generate's onToken callback (Engine.swift:922, :1024): called on the calling
 * thread with each token as it is delivered; return 0 to stop the request. */
typedef int (*ill_token_fn)(int32_t token, void* user);

/* ill_generate with a per-token callback. When the callback returns 0 the request stops:
 * the steps already queued leave at once (Engine.swift:1032-1036), the K/V cache keeps
 * the prompt and the delivered tokens but the last, and n_out counts the delivered tokens. */
ILL_API int ill_generate_cb(ill_engine* e, const int32_t* toks, int ntok, int max_new, int chunk,
                    int32_t* out, int* n_out, float* logits_out, ill_token_fn on_token, void* user);

/* The host's stop for passes already launched (Engine.swift:1032-1036 writes the State's
 * done flag into shared memory). The word lives in pinned host memory; the commit of every
 * pass reads it (the read is issued when the pass starts): a pass that sees it commits
 * nothing and sets the device State's done flag, so every pass queued behind it leaves at
 * its header. A pass whose commit read the word before the call completes normally.
 * ill_set_state clears it. Safe to call from another thread while a generate call or a
 * launched graph runs. */
ILL_API int ill_stop(ill_engine* e);

/* ---- Speculative decoding with on-device drafting (k_commit_spec, Shaders.swift:246-418) ----
 * With the State's tspec = T > 1, every commit of a prefill or verify pass is speculative: it
 * accepts the longest prefix of the pass's drafts that equals the rows' argmaxes, commits
 * those tokens, then drafts up to T - 1 tokens for the next pass on the device
 * (self-repetition of the output, then the n-gram table, then prompt lookup;
 * Shaders.swift:367-412) and sets up that pass as a chain over [last token, drafts...].
 * The tokens committed equal plain greedy decoding's (every row's logits equal a 1-row
 * step's, bit for bit). The State's passes / accepted fields count passes and accepted
 * drafts (Engine.swift:959). */

/* Engine.loadNGram (Engine.swift:747-753): an n-gram draft table in the NGramTable layout
 * (NGram.swift:1-59): 2^20 slots of {u64 key, i32 next, u16 count, u16 total}, 16 MiB.
 * table NULL (or bytes 0) unloads it. */
ILL_API int ill_load_ngram(ill_engine* e, const void* table, int64_t bytes);

/* The prompt-lookup context of the drafter (promptRecent, Engine.swift:125, :939-942): the
 * last <= 256 of the request's prompt tokens. ill_generate_spec sets it itself. */
ILL_API int ill_set_prompt(ill_engine* e, const int32_t* toks, int n);

/* One verify pass over the rows the last speculative commit drafted (encodeSpecPass /
 * encodeWidePass + k_commit_spec, Engine.swift:524-579), launched and waited for. */
ILL_API int ill_spec_pass(ill_engine* e, int write_logits);

/* Record `npasses` such passes into one hipGraph (Engine.swift:991-1013 encodes them the
 * same way for every format): each pass takes its rows from the commit before it, so the
 * graph chains verify passes without the host; passes after the stop flag early-exit. q4
 * passes run on the pass-kernel instantiation of the State's tspec rows; q8 and f16 passes
 * on the layer-by-layer kernels launched for as many rows, of which the rows a pass does
 * not hold are computed and never committed. ill_launch_graph replays it. */
ILL_API int ill_capture_spec(ill_engine* e, int npasses);

/* Engine.generate with speculation on (Engine.swift:922-1038): prefill, then verify passes
 * of up to `rows` (2..16) rows, in captured graphs of `chunk` passes (every format), while
 * polling out_tokens. adaptive != 0 chooses each pass's
 * shape from the accepted drafts per pass (Engine.nextPassShape, :888-898, with thresholds
 * from this engine's pass costs, which grow with the kernel's row count): the configured
 * shape while at least 2.4 are accepted, 4-row chains while at least 1.6 are (back to the
 * configured shape at 2.2), else one-row passes with a 4-row probe after 16 passes (the
 * gap doubles, up to 128, after each probe that fails). A shape is judged on its own
 * passes, after two of them (one that accepted nothing), with one of them in flight at a
 * time until then; a change to one-row passes cuts the pending drafted pass to its first
 * row. The tokens are those of greedy decoding in every case.
 * out / n_out as for ill_generate; stats (optional, [2]) receives the passes and accepted
 * drafts of the request. */
ILL_API int ill_generate_spec(ill_engine* e, const int32_t* toks, int ntok, int max_new, int rows, int chunk, int adaptive,
                      int32_t* out, int* n_out, int32_t* stats);

/* ---- Learned drafter (ILDraft.swift:1-209, k_ildraft Shaders.swift:421-872) ----------------
 * A table in the ILDRAFT1 format (tools/draft/ildraft.py:16-53) scores the candidates of the
 * n-gram statistics, self-repetition, prompt lookup, the request's TF-IDF neighbours'
 * outputs and the copy candidates with 53 features and a small MLP; a drafting kernel runs
 * it after each speculative commit and proposes the next pass: a chain of up to
 * chain_rows - 1 tokens, or a best-first tree of up to tree_budget tokens (8 children per
 * expansion) verified in one tree pass. Speculation never changes the tokens committed.
 *
 * ill_ildraft_open (ILDraft.init, :38-84): reads and checks a table (NULL on error, see
 * ill_last_error). ill_ildraft_prepare (ILDraft.prepare, :110-208): the per-request context
 * from the user prompt's ids inside the chat template, its text and the tokenizer
 * (`encode` writes the ids of a text into ids[0..cap) and returns their count; NULL: no
 * space-variant candidates). ill_ildraft_request copies the prepared context (the
 * IllDraftReq layout of instantllm_amd/csrc/ill_ildraft.h) and returns its size in bytes. */
typedef struct ill_ildraft ill_ildraft;
typedef int (*ill_encode_fn)(void* user, const char* text, int32_t* ids, int cap);
ILL_API ill_ildraft* ill_ildraft_open(const char* path);
ILL_API void ill_ildraft_close(ill_ildraft* d);
ILL_API int ill_ildraft_prepare(ill_ildraft* d, const int32_t* prompt, int n, const char* text, ill_encode_fn encode, void* user);
ILL_API int64_t ill_ildraft_request(const ill_ildraft* d, void* out, int64_t bytes);

/* Engine.loadLearnedDrafter (Engine.swift:901-904): loads a table into the engine. */
ILL_API int ill_load_ildraft(ill_engine* e, const char* path);

/* Engine.setDraftContext (Engine.swift:908-913): prepares the next ill_generate_spec
 * request's drafter context (at once, on the CPU). That call then drafts with the learned
 * drafter (Engine.swift:950-956) and consumes the context. */
ILL_API int ill_set_draft_context(ill_engine* e, const int32_t* prompt, int n, const char* text, ill_encode_fn encode, void* user);

/* Engine.useLearned / learnedT / learnedTree (Engine.swift:871-880): use != 0 lets a
 * prepared context switch ill_generate_spec to the learned drafter; its passes are chains
 * of chain_rows (2..16) rows, or with tree_budget > 0 trees of min(tree_budget, 15) drafts
 * (passes of that + 1 rows; with ill_generate_spec's `adaptive` these are its configured
 * shape). Defaults 1, 8, 15. */
ILL_API int ill_set_learned(ill_engine* e, int use, int chain_rows, int tree_budget);

/* The pass the last speculative commit set up (no reference counterpart: inspection for
 * tests and tools): info = [mode (1 chain, 2 tree), rows, commit, drafting still pending];
 * toks [16] the rows' tokens; tree [65] the tree buffer (Shaders.swift:23-30 layout). */
ILL_API int ill_pending_pass(ill_engine* e, int32_t info[4], int32_t toks[16], int32_t tree[65]);

/* ---- Prefix reuse across requests (Engine.swift:788-838, :929-933, :1029-1031) ----------
 * ill_generate / ill_generate_spec keep the tokens whose K/V stay valid after the call (the
 * prompt and every generated token but the last); the next call prefills only the part of
 * its prompt after the longest common prefix (at least one token). Any pass or K/V write
 * launched outside those calls forgets the cached tokens.
 * ill_prefix_info: the cached token count and the tokens the last generate call prefilled.
 * ill_save_prefix (Engine.savePrefix): writes the K/V of the first n cached tokens (toks
 * must be that prefix) to `path`: [u64 key: magic, model file size, mtime s, mtime ns,
 * max_context][u64 n][n x i32 tokens][K][V], K and V as [layer][kv head][n][64] f16.
 * ill_load_prefix (Engine.loadPrefix): loads such a file if it was saved for this model
 * file and context (else ILL_E_FILE), makes its tokens the cached prefix and returns them
 * in toks (max_toks entries; NULL to skip) and their count in n_out. */
ILL_API int ill_prefix_info(ill_engine* e, int* cached, int* last_prefill);
/* Engine.truncateCache (Engine.swift:850-853): forget the cached K/V beyond the first n
 * tokens (0 clears the cache). A reused prefix changes where the prompt's last tokens are
 * computed (its K/V come from the earlier request's passes), so a near tie can resolve
 * differently than from a cold cache; callers comparing runs clear it first. */
ILL_API int ill_truncate_cache(ill_engine* e, int n);
ILL_API int ill_save_prefix(ill_engine* e, const char* path, const int32_t* toks, int n);
ILL_API int ill_load_prefix(ill_engine* e, const char* path, int32_t* toks, int max_toks, int* n_out);

/* Timing (Engine.profile / gpuTime, Engine.swift:621-729): GPU milliseconds of `iters`
 * replays of the captured graph, measured with HIP events on the engine's stream. */
ILL_API int ill_time_graph(ill_engine* e, int iters, float* ms);

/* GPU milliseconds of the most recent single pass (prefill chunk, decode step or verify
 * pass launched through the functions above), from HIP events around its kernel. */
ILL_API int ill_last_pass_ms(ill_engine* e, float* ms);

/* Per-workgroup timeline of the pass kernel (the persistent-kernel counterpart of
 * Engine.profile's per-kernel times): when on, thread 0 of every workgroup stores the
 * 100 MHz device clock at points of its role in every layer l (slot 16 l + k: k = 0 role
 * start, 1 input ready, 11 done, 2-10 and 12-15 role-specific intermediate points), and
 * of the lm_head and commit tail (slots 480 + k). Unreached slots stay 0.
 * ill_trace_read copies [256][slots] u64 values of the last pass and returns `slots`. */
ILL_API int ill_trace_enable(ill_engine* e, int on);
ILL_API int ill_trace_read(ill_engine* e, uint64_t* out, int* slots);

/* Stand-alone q4 GEMV, the decode step's matrix-vector product measured on its own
 * The reference has no separate entry for it: it times the same
 * kernels (q4_chunk_norm / q_rows, k_lm_head_T; Shaders.swift:1001-1185, :1327-1364) inside
 * Engine.profile (Engine.swift:639-729). codes [rows][K/2] and scales [rows][K/64] (f16
 * scale | f16 min << 16) are the .ill q4 layout; `copies` device copies of the weights are
 * rotated through so that repeated runs stream from HBM rather than the 256 MB MALL.
 * ill_gemv_run: y = W * rmsnorm(x) * gamma (gamma NULL: y = W * x), `iters` timed runs;
 * y (host [rows], optional) and argmax (host, optional: lowest index of the maximum,
 * which also enables the argmax epilogue) are from the last run. */
typedef struct ill_gemv ill_gemv;
ILL_API int ill_gemv_create(int rows, int K, const uint8_t* codes, const uint32_t* scales, int copies, ill_gemv** out);
ILL_API int ill_gemv_run(ill_gemv* g, const float* x, const float* gamma, int iters, float* y, int32_t* argmax, float* us_per_iter);
ILL_API int ill_gemv_info(const ill_gemv* g, int* slices, int* blocks_per_slice, int64_t* bytes_per_copy);

/* No counterpart in the reference: ill_gemv_run for callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc). One product on weight copy `copy` of g, enqueued on `stream` (a hipStream_t;
 * NULL: g's own stream) and not waited for. x [K], gamma [K] (NULL: plain input), y [rows]
 * and argmax (one int32) are device pointers owned by the caller; y may be NULL when
 * argmax is not (the product then lives in the library's per-GPU scratch array, at most
 * 262144 rows; larger products need a y buffer). The call allocates nothing: the argmax
 * keys live in that same fixed scratch array, shared by every call on the GPU, so calls
 * that overlap on one GPU race. Same arithmetic and results as ill_gemv_run. */
ILL_API int ill_gemv_run_noalloc(ill_gemv* g, int copy, const float* x, const float* gamma, float* y, int32_t* argmax, void* stream);
ILL_API int ill_gemv_destroy(ill_gemv* g);

/* ---- Paged cache: several sequences at once (no counterpart in the reference) --------------
 * Operators on device buffers for programs that serve many requests: keys and values live in
 * pages of a cache that the caller owns, and a batch names each sequence's pages. Like
 * ill_gemv_run_noalloc, the calls take device pointers, enqueue on the caller's `stream` (a
 * hipStream_t; NULL: the device's default stream), allocate nothing, wait for nothing and can
 * be captured into a graph.
 *
 * A handle holds a model's geometry: `heads` query heads over `kv_heads` key/value heads (query
 * head h reads key/value head h / (heads / kv_heads)) of `head_dim` 64 or 128; a cache of type
 * ILL_F16 or ILL_BF16 in pages of `page_size` positions (a power of two, 16 .. 1024). Element
 * (page, slot, head, dim) of either cache is at page * page_stride + slot * slot_stride +
 * head * head_stride + dim elements (all 0: [pages][page_size][kv_heads][head_dim]); strides are
 * multiples of 8, slot_stride at most 2^24. The rotation turns the first `rotary_dim` dims of a
 * head (a multiple of 16; 0: none) by position * rope_base^(-2 i / rotary_dim), pairing dim i
 * with i + rotary_dim / 2, or with interleaved != 0 dims 2 i and 2 i + 1. norm_eps belongs to the head norms; scale
 * multiplies the scores (0: 1 / sqrt(head_dim)). A handle belongs to the GPU that was current
 * when it was created; one thread at a time calls on it.
 * dtype ILL_F16 | ILL_MXF8 or ILL_BF16 | ILL_MXF8: a cache of microscaled 8-bit values (ILL_MXF8 below) for queries and outputs
 * of the other type, 33 bytes for 32 values. A page is [kv_heads][page_size][head_dim] codes followed by [kv_heads][page_size]
 * [head_dim / 32] powers; page_stride is the bytes from one page to the next (a multiple of 16; 0: no gap), slot_stride and
 * head_stride are 0. ill_paged_append quantises each head's blocks of 32 as ill_mx_quantize does, from the float32 values; an infinity
 * or NaN makes its block NaN. ill_paged_attend takes the cache's values as values of the handle's type: bf16 has an exact place for
 * all but the least of them, f16 rounds below 2^-14 and is infinite past 65504. Everything else holds for either kind of cache.
 * Attention that is split over the keys joins its parts through a workspace, one of `streams`
 * that the handle holds (0: 8; 11 MB each at head size 64, 22 at 128). Each stream that calls
 * come on takes one, and so does each capture of a stream: calls on different streams, and
 * graphs, may run at the same time. (hipStreamPerThread, a different stream in each thread, is
 * refused.) What is enqueued on one stream, or captured on one stream in one capture, shares a
 * workspace: such a graph is instantiated once. A call that would need one more is refused.
 * ill_paged_bind makes a stream's calls, captured or not, take workspace 0 .. streams - 1
 * from now on: a program that launches its graphs in order captures all of them on streams
 * bound to one workspace. What was enqueued or captured on streams of one workspace must not
 * run at the same time. A workspace that an unbound stream's calls hold is refused, and a
 * second one for a stream. Workspace -1: the stream is bound no more, and the workspaces that its calls and captures have taken
 * are free; called when nothing that came on the stream will run any more, also before a
 * stream is destroyed (a later one may get its address). ill_paged_release does so for all
 * streams. */
enum { ILL_F32 = 0, ILL_F16 = 1, ILL_BF16 = 2, ILL_MXF8 = 8, ILL_MXF4 = 16 };
typedef struct ill_paged ill_paged;
typedef struct {
  int32_t dtype, heads, kv_heads, head_dim, page_size, rotary_dim, interleaved, streams;
  int64_t page_stride, slot_stride, head_stride;
  double rope_base;
  float norm_eps, scale;
} ill_paged_desc;
ILL_API int ill_paged_create(const ill_paged_desc* desc, ill_paged** out);
ILL_API int ill_paged_destroy(ill_paged* p);
ILL_API int ill_paged_bind(ill_paged* p, void* stream, int workspace);
ILL_API int ill_paged_release(ill_paged* p);

/* A batch. lens, table and row0 are device arrays that the kernels read when they run, so a
 * captured call follows what they then hold. lens [seqs]: the positions of each sequence, its
 * new rows included (below 0 counts as 0). table [seqs][table_stride], table_width entries used:
 * the page of positions i * page_size .. in entry i; entries behind a sequence's last position
 * are not read. row0 [seqs + 1]: ascending; sequence s has the new rows row0[s] ..
 * row0[s + 1] - 1, which stand at its last positions; NULL: row s is sequence s's only one.
 * rows: rows of the buffers (the ones that are no sequence's are left alone). max_rows: the most
 * new rows that a sequence has, if known (0: unknown; a hint for the launch only: without it
 * single rows that come with row0 are launched with prompts' workgroups too, which end at once;
 * 200 rows in a window 27.5 in place of 24.3 us). pages: pages of the cache. A page number outside 0 .. pages - 1 is not followed: its positions are neither
 * written nor seen, and so are positions past table_width pages or below 0. Pages may be shared
 * for reading. rows x heads is at most 2^26, seqs x heads at most 2^22, seqs at most 2^14 (from
 * a thousand on a call's time grows with their square: 1024 with 2 key/value heads 42 us, 4096 320). */
typedef struct {
  int32_t seqs, table_width;
  int64_t table_stride, rows, max_rows, pages;
  const int32_t *lens, *table, *row0;
} ill_paged_batch;

/* New rows into the cache. q, k, v: rows of heads x head_dim (kv_heads x head_dim) values of
 * type `dtype` (ILL_F32, or the handle's), row r at r * stride elements; parts of one fused
 * product will do. q NULL: keys and values only. To each head's x: x + bias (bias [(heads + 2
 * kv_heads) x head_dim], q then k then v), then for q and k x / sqrt(mean(x^2) + norm_eps) *
 * q_norm (k_norm) [head_dim], then the rotation by the row's position (positions [rows]: by
 * these instead), computed in float32 from angles in float64 and rounded once. NULL leaves a
 * step out. Keys and values go to their slots, queries to q_out (the handle's type; q itself
 * will do where type and stride agree). Two rows of one batch must not share a slot, and
 * q_out and the caches overlap nothing else that the call reads. Buffers
 * and caches are aligned to 16 bytes, strides are multiples of 8 elements (float32: 4). */
typedef struct {
  const void *q, *k, *v;
  void* q_out;
  int64_t q_stride, k_stride, v_stride, q_out_stride;
  const float *bias, *q_norm, *k_norm;
  const int32_t* positions;
  int32_t dtype, reserved;
} ill_paged_rows;
ILL_API int ill_paged_append(ill_paged* p, const ill_paged_batch* batch, const ill_paged_rows* rows, void* k_cache, void* v_cache,
                             void* stream);

/* Attention of the new rows over the cache (what ill_paged_append has written included): the
 * row at position p sees the positions j <= p with j > p - window (window 0: all of them) or
 * j < sinks. out [rows][heads x head_dim], row r at r * out_stride, of type out_dtype (the
 * handle's, or ILL_F32): the values weighted by the softmax of the scaled scores; zeros for a row
 * that sees nothing (or whose scores are all -inf). Sums are float32, of weights of at most 1 for a
 * bf16 cache (an f16 cache's values cannot overflow them). For 16-bit outputs the weights are rounded once to
 * the handle's type before they multiply the values, each by up to 2^-8 (bf16) or 2^-11 (f16) of itself; for
 * float32 outputs they keep 22 bits and more. q [rows][heads x head_dim] is of the
 * handle's type; out overlaps nothing that the call reads. What a row does not see never reaches it, infinities and NaN included. A value
 * that is infinite or NaN reaches every row that sees it, however small its weight: the output
 * is that infinity, or NaN where the row also sees a NaN or the other one; unless all of the
 * row's scores are -inf, or one is +inf or NaN (the row is then NaN). */
ILL_API int ill_paged_attend(ill_paged* p, const ill_paged_batch* batch, const void* q, int64_t q_stride, const void* k_cache,
                             const void* v_cache, int window, int sinks, void* out, int64_t out_stride, int out_dtype, void* stream);

/* The batch's rows out of the cache, where ill_paged_append would put them: keys to k, values to v, rows of kv_heads x head_dim
 * values, row r at r * stride, of type out_dtype (the handle's, or ILL_F32), as the cache holds them. With row0 over all of a sequence's
 * positions that is the whole sequence. Zeros for a row without a place in the cache; rows that are no sequence's are left alone.
 * k and v are aligned to 16 bytes, strides multiples of 8 elements (float32: 4); they overlap nothing else that the call reads or writes. */
ILL_API int ill_paged_read(ill_paged* p, const ill_paged_batch* batch, const void* k_cache, const void* v_cache, void* k, int64_t k_stride,
                           void* v, int64_t v_stride, int out_dtype, void* stream);

/* ---- Microscaled rows: quantisation and products for batches (no counterpart in the reference) ----
 * A microscaled row is blocks of 32 values that share a power of two. A block's byte e stands for 2^(e - 127), 255
 * for a block of NaN. Codes are e4m3 (ILL_MXF8: one byte, up to 448) or e2m1 (ILL_MXF4: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
 * negatives; two to a byte, the first in the low four bits). A matrix of rows is two arrays: codes [rows][cols or cols / 2] and powers
 * [rows][cols / 32], both without gaps and aligned to 16 bytes; cols is a multiple of 32.
 * Like the calls on a paged cache these take device pointers, enqueue on `stream` (a hipStream_t; NULL: the current device's
 * default stream), allocate nothing, wait for nothing, keep nothing and can be captured into a graph. They run on the GPU that the stream belongs to.
 *
 * ill_mx_quantize: x [rows][cols] of type `dtype`, row r at r * x_stride elements (a multiple of 8, float32: 4; x aligned to 16
 * bytes). A block's power is floor(log2(the largest size in it)) - 8 (ILL_MXF4: - 2), at least 2^-127; its values divided by it
 * are rounded to nearest, ties to even, and end at +-448 (+-6). A block that holds an infinity or NaN becomes NaN (codes 0).
 * ill_mx_dequantize: the values, rounded to `dtype` where they have no exact place in it. Up to 2^34 values a call. What a call writes
 * overlaps nothing that it reads. */
ILL_API int ill_mx_quantize(int format, int dtype, const void* x, int64_t x_stride, int64_t rows, int64_t cols, void* codes, void* powers, void* stream);
ILL_API int ill_mx_dequantize(int format, int dtype, const void* codes, const void* powers, int64_t rows, int64_t cols, void* y, int64_t y_stride,
                              void* stream);

/* y[r][c] = the sum over k of x[r][k] w[c][k], plus bias[c] (NULL: none): x [rows][inner] of format x_format, the matrix w
 * [cols][inner] of format ILL_MXF4, both as ill_mx_quantize writes them. y: row r at r * y_stride elements of type y_dtype, rounded
 * once; aligned to its type (to 16 bytes, with strides of whole 16 bytes, it is stored fastest). inner: a multiple of 32 up to 2^20
 * (from 17 rows on, multiples of 128 are up to 1.5 times as fast); cols up to 2^24, rows up to 2^26, rows x cols up to 2^32.
 * Sums are float32's, in an order that depends on the sizes and types alone. With x of format ILL_MXF8 and a 16-bit y they are the
 * matrix units' own: of eight neighbouring values' products (the first eight, the next, ...) each loses less than 2^-12 of the largest
 * one's size, and the largest nothing. Before it is rounded an output is so off by 7 x 2^-12 of the sum of its products' sizes at most;
 * by the 2-norm of all outputs by up to 1e-5 for normal values, and 2e-5 to 7e-5 where every 61st is fifty times as large or codes and
 * powers have evenly spread exponents. For a float32 y of such x both operands are multiplied as bf16 values: not cut, but values below
 * 2^-126 may count as 0, and ones past bf16's range as infinite. A NaN block makes every output that it belongs to NaN. y overlaps
 * nothing that the call reads. */
ILL_API int ill_mx_product(int x_format, const void* x, const void* x_powers, const void* w, const void* w_powers, int64_t rows, int64_t cols,
                           int64_t inner, const float* bias, int y_dtype, void* y, int64_t y_stride, void* stream);

/* The converter's quantizers (Converter.quantizeQ4Raw / quantGroup and quantizeQ8,
 * Sources/Engine/Convert.swift:252-370), host code that needs no GPU. w is a row-major
 * float32 [rows][cols] matrix; `threads` CPU threads split the rows (any count gives the
 * same bytes).
 * q4: packed [rows][cols/2] codes (column 2j in the low nibble of byte j) and sb
 * [rows][cols/64][2] f16 bits (scale, bias): per 64 columns the clipped-range search with a
 * least-squares refit that keeps the lowest squared error after f16 rounding.
 * q8: codes [rows][cols] and scales [rows][cols/group] f16 bits, group 32 (the reference) or
 * 64: symmetric, scale = f16(amax/127) raised one ulp when a code would leave -127..127. */
ILL_API int ill_quantize_q4(const float* w, int64_t rows, int cols, uint8_t* packed, uint16_t* sb, int threads);
ILL_API int ill_quantize_q8(const float* w, int64_t rows, int cols, int group, int8_t* codes, uint16_t* scales, int threads);

/* The tokenizer (Sources/Tokenizer: Tokenizer.swift, Core.swift; host code, no GPU):
 * Qwen2 byte-level BPE, equal to Hugging Face `tokenizers` on the same tokenizer.json.
 * `python -m instantllm_amd.tokenizer compile tokenizer.json out.iltk` writes the file
 * (Tokenizer.compile, Compile.swift:14-371) that ill_tok_open maps (Tokenizer(path:),
 * Tokenizer.swift:57-117). ill_tok_info: ids in total (vocabulary and added tokens), and the
 * ids of <|im_start|>, <|im_end|>, <|endoftext|> (-1: absent).
 * ill_tok_encode: `specials` 0 is Tokenizer.encode (:150-152, no added-token matching),
 * 1 is encodeWithSpecials (:154-158, added tokens matched leftmost-longest on the raw text);
 * ill_tok_encode_chat is encodeChat (:160-183, the chat template around system and user);
 * ill_tok_decode is decode (:275-295: the tokens' bytes, ill-formed UTF-8 replaced by U+FFFD,
 * ids without a token skipped); ill_tok_token_bytes is tokenBytes (:266-271, valid while
 * the tokenizer is open); ill_tok_normalize and ill_tok_pretokenize are normalize and
 * preTokenize (:299-323: the NFC text, and the end offsets of the pieces of an NFC text).
 * Text arguments are UTF-8 of the given byte length (anything else: ILL_E_ARG). Output
 * buffers hold `cap` entries; the count or length is always written, and when it exceeds
 * cap the call fails with ILL_E_ARG. ill_tok_encode_cb is an ill_encode_fn over an ill_tok
 * (the `user` argument): encodeWithSpecials of a NUL-terminated text, the first cap ids
 * written and their whole count returned (0 for text that is not UTF-8). */
typedef struct ill_tok ill_tok;
ILL_API int ill_tok_open(const char* path, ill_tok** out);
ILL_API int ill_tok_close(ill_tok* t);
ILL_API int ill_tok_info(const ill_tok* t, int32_t info[4]);
ILL_API int ill_tok_encode(const ill_tok* t, const char* text, int64_t len, int specials, int32_t* ids, int64_t cap, int64_t* n);
ILL_API int ill_tok_encode_chat(const ill_tok* t, const char* system, int64_t slen, const char* user, int64_t ulen, int32_t* ids,
                                int64_t cap, int64_t* n);
ILL_API int ill_tok_decode(const ill_tok* t, const int32_t* ids, int64_t n, char* out, int64_t cap, int64_t* len);
ILL_API int ill_tok_token_bytes(const ill_tok* t, int32_t id, const char** bytes, int64_t* len);
ILL_API int ill_tok_normalize(const ill_tok* t, const char* text, int64_t len, char* out, int64_t cap, int64_t* olen);
ILL_API int ill_tok_pretokenize(const ill_tok* t, const char* text, int64_t len, int64_t* ends, int64_t cap, int64_t* n);
ILL_API int ill_tok_encode_cb(void* user, const char* text, int32_t* ids, int cap);

#ifdef __cplusplus
}
#endif
#endif
