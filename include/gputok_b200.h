/*
 * gputok_b200.h -- C ABI of the B200-native greedy byte-level BPE tokenizer.
 *
 * This is the drop-in boundary for the reference's `GpuTokenizer` class
 * (gputok_binding.cu:650-1011, exported to Python at :1015-1065).  Every entry
 * point is `extern "C"`, takes plain pointers and sizes, returns an `int`
 * status (GTK_OK == 0) and never throws or exits; the message of the last
 * failure is available from gtk_last_error() / gtk_global_error().
 *
 * Semantics shared by all encode entry points (reference:
 * gputok_binding.cu:704-752, 823-836):
 *   - a batch is `n_texts` byte strings laid back to back in one buffer;
 *     text t is bytes[text_offsets[t] .. text_offsets[t+1]), text_offsets[0]
 *     must be 0 and the array non-decreasing;
 *   - every text is cut into chunks of `chunk_tokens` bytes (the last chunk of
 *     a text may be shorter, an empty text has no chunk); chunks are tokenised
 *     independently with the greedy rule (globally lowest merge rank, left-most
 *     occurrence, one merge at a time until no adjacent pair is mergeable:
 *     bpe_merge_cpu_greedy, gputok_blockbpe.cu:248-300);
 *   - token ids live in the reference's id space: ids 0..255 are the byte
 *     values, merge number r (0-based line of merges.txt after the header)
 *     creates id 256+r for a well-formed table (build_vocab_and_merges,
 *     gputok_blockbpe.cu:178-236);
 *   - the result is packed: all ids of the batch back to back in chunk order,
 *     int64 offsets per chunk and per text.
 */
#ifndef GPUTOK_B200_H
#define GPUTOK_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define GTK_API __attribute__((visibility("default")))
#else
#define GTK_API
#endif

/* status codes */
enum {
  GTK_OK               = 0,
  GTK_ERR_INVALID_ARG  = 1, /* e.g. chunk_tokens <= 0 (std::invalid_argument, gputok_binding.cu:661-663) */
  GTK_ERR_IO           = 2, /* merges file unreadable or empty (std::runtime_error, :153-161) */
  GTK_ERR_CUDA         = 3, /* a CUDA runtime call failed (the reference prints and exit()s, :24-30) */
  GTK_ERR_CAPACITY     = 4, /* a caller-provided output buffer is too small */
  GTK_ERR_TABLE        = 5, /* the entry point does not serve this merge table (see gtk_create) */
  GTK_ERR_NO_DEVICE    = 6, /* GPU entry point called on a host-only handle */
  GTK_ERR_KERNEL       = 7, /* a kernel reported an internal inconsistency through its status word */
  GTK_ERR_MEMORY       = 8  /* the host has no memory left (std::bad_alloc in the reference) */
};

/* which merge kernel serves the call */
enum {
  GTK_MODE_OPT  = 0, /* GpuTokenizer::tokenize_batch               (gputok_binding.cu:704-846) */
  GTK_MODE_BASE = 1, /* GpuTokenizer::tokenize_batch_blockbpe_base (gputok_binding.cu:850-989) */
  GTK_MODE_LOCALMIN = 2 /* the reference's OTHER rule on the GPU: bpe_merge_kernel_optimized (gputok_binding.cu:290-414),
                           per chunk, at most max_iters passes; not greedy Algorithm 1 -- offered for timing and
                           behaviour comparisons with the reference's tokenize_batch only */
};

/* merge rule of the host reference entry point */
enum {
  GTK_RULE_GREEDY   = 0, /* bpe_merge_cpu_greedy, per chunk (gputok_blockbpe.cu:248-300) */
  GTK_RULE_LOCALMIN = 1  /* bpe_merge_cpu, whole text, max_iters passes (gputok_binding.cu:200-270, 992-1003) */
};

typedef struct gtk_tokenizer gtk_tokenizer;

typedef struct gtk_table_info {
  int32_t  vocab_size;       /* number of token ids (50 256 for GPT-2 merges.txt) */
  int32_t  num_merges;       /* distinct (left,right) pairs in the table */
  uint32_t max_rank;         /* highest rank present */
  uint32_t hash_capacity;    /* slots of the pair table: 65 536 buckets of four */
  uint32_t hash_overflow_entries; /* pairs whose bucket was full (side table, second load) */
  uint32_t hash_bytes;       /* bytes of the pair table in HBM */
  int32_t  monotone;         /* 1: every merge has a higher rank than the merges that create its parts */
  int32_t  merged_is_256_plus_rank; /* 1: merged id == 256 + rank for every merge */
  int32_t  byte_ids_identity;       /* 1: id of byte b == b for all 256 bytes */
  int32_t  adj_bigrams;      /* byte bigrams that occur inside at least one merge result */
  int32_t  chunk_tokens;
  int32_t  max_iters;
  int32_t  device;           /* CUDA device ordinal, -1 for a host-only handle */
  int32_t  sm_count;
  int32_t  whole_segment_entries;   /* vocabulary strings (2..16 bytes) answered by one table probe */
  uint32_t whole_segment_dropped; /* qualifying strings that found no place (they are merged instead) */
} gtk_table_info;

/* Library version string. */
GTK_API const char* gtk_version(void);

/* Message of the last failure that had no handle to attach to (gtk_create). Thread-local. */
GTK_API const char* gtk_global_error(void);

/* Replaces GpuTokenizer::GpuTokenizer(merges_path, chunk_tokens, max_iters)
 * (gputok_binding.cu:652-701): parses merges.txt, rebuilds the vocabulary,
 * builds the merge-rank hash table, the byte-pair rank table and the
 * never-merge bigram bitmap and uploads them to `device`.
 * chunk_tokens <= 0 -> GTK_ERR_INVALID_ARG; max_iters <= 0 -> 50 (as :664-666).
 * device == -1 builds a host-only handle: the GPU entry points then return
 * GTK_ERR_NO_DEVICE (there is no CPU fallback); gtk_encode_cpu still works.
 * Any merges file the reference accepts is accepted (it carries int32 ids and a 64-bit pair key,
 * gputok_blockbpe.cu:139-157).  The fast kernels hold ids and ranks in 16 bits; a table with ids
 * >= 65535 or ranks >= 65534 (beyond roughly 65 000 merges; GPT-2 has 50 000) is served, for both
 * GTK_MODE_OPT and GTK_MODE_BASE, by a 32-bit one-CTA-per-chunk kernel with the same results at
 * the speed of the literal design.  For such a table GTK_MODE_LOCALMIN and
 * gtk_encode_chunks_noalloc return GTK_ERR_TABLE. */
GTK_API int gtk_create(const char* merges_path, int chunk_tokens, int max_iters, int device,
                       gtk_tokenizer** out);

/* Replaces the destructor of GpuTokenizer (frees the table and all arenas). */
GTK_API void gtk_destroy(gtk_tokenizer* h);

GTK_API const char* gtk_last_error(const gtk_tokenizer* h);

GTK_API int gtk_table_info_get(const gtk_tokenizer* h, gtk_table_info* out);

/* Replaces tokenize_batch (mode GTK_MODE_OPT, gputok_binding.cu:704-846) and
 * tokenize_batch_blockbpe_base (mode GTK_MODE_BASE, :850-989) for HOST input.
 * Copies the batch to the device (fastest from pinned memory, see
 * gtk_pinned_alloc), runs chunker -> merge kernel -> output scan/pack, copies
 * ids and offsets back into pinned buffers owned by the handle.
 * *kernel_ms (optional) receives the device time of the kernel pipeline, from
 * the first kernel of the call to the end of the last (the reference's event
 * pair, :790-805; see gtk_last_stage_ms).  Results stay valid until the next
 * call on the handle; read them with gtk_result_sizes/_view/_copy.
 * An empty batch or a batch of empty texts is not an error: 0 ids, 0 chunks.
 * Small batches (up to 8 KiB and 1024 texts, GTK_MODE_OPT) run as one kernel that reads the text from and
 * writes the results to mapped page-locked memory; the call returns when the kernel's completion mark has
 * arrived there (its last store, behind a system-wide fence), which is when the results are complete -- the
 * stream may still be retiring the kernel for a few microseconds.  *kernel_ms is then the kernel's own
 * measurement of its duration. */
GTK_API int gtk_encode(gtk_tokenizer* h, int mode, const uint8_t* bytes, const int64_t* text_offsets,
                       int64_t n_texts, float* kernel_ms);

/* The same for strings that lie anywhere: text t is texts[t][0 .. text_offsets[t+1] - text_offsets[t]).  They are gathered
 * into page-locked memory inside the call, by up to three helper threads of the handle's when there is much to gather,
 * while what has been gathered is on its way to the device. */
GTK_API int gtk_encode_strings(gtk_tokenizer* h, int mode, const uint8_t* const* texts, const int64_t* text_offsets,
                               int64_t n_texts, float* kernel_ms);

/* Replaces tokenize_batch_cpu (gputok_binding.cu:992-1003): host-only
 * reference tokenizer.  GTK_RULE_GREEDY (default of the Python surface) runs
 * the greedy rule per chunk; GTK_RULE_LOCALMIN reproduces the reference
 * method's own rule on the un-chunked text.  Never used as a fallback. */
GTK_API int gtk_encode_cpu(gtk_tokenizer* h, int rule, const uint8_t* bytes, const int64_t* text_offsets,
                           int64_t n_texts);

/* Sizes of the result of the last gtk_encode / gtk_encode_cpu. */
GTK_API int gtk_result_sizes(const gtk_tokenizer* h, int64_t* n_ids, int64_t* n_chunks, int64_t* n_texts);

/* Zero-copy view of the last result (replaces the unflatten loop,
 * gputok_binding.cu:823-836): ids[n_ids], text_id_offsets[n_texts+1]
 * (text t owns ids[text_id_offsets[t] .. text_id_offsets[t+1])),
 * chunk_id_offsets[n_chunks+1].  Pointers are owned by the handle. */
GTK_API int gtk_result_view(const gtk_tokenizer* h, const int32_t** ids, const int64_t** text_id_offsets,
                            const int64_t** chunk_id_offsets);

/* Copy of the last result into caller buffers (any of them may be NULL). */
GTK_API int gtk_result_copy(const gtk_tokenizer* h, int32_t* ids, int64_t ids_capacity,
                            int64_t* text_id_offsets, int64_t* chunk_id_offsets, int64_t chunk_capacity);

/* Device-resident variant of gtk_encode for callers that keep text and ids in
 * HBM (replaces the kernel launch section, gputok_binding.cu:790-805, together
 * with the host chunk/flatten loops :718-752 that now run on the device).
 * d_bytes (16-byte aligned for full speed), d_text_offsets[n_texts+1] (int64),
 * d_out_ids[out_capacity] and d_out_chunk_offsets[chunk_capacity] (>= number
 * of chunks + 1, may be NULL) are device pointers on the handle's device.
 * d_text_offsets[0] is 0; bytes from d_text_offsets[n_texts] to n_bytes belong to no text and yield no ids.
 * *n_ids / *n_chunks are host outputs.  Synchronous on return.  GTK_ERR_CAPACITY
 * if a buffer is too small: nothing is written past a capacity, what was
 * written before the error is unspecified. */
GTK_API int gtk_encode_device(gtk_tokenizer* h, int mode, const uint8_t* d_bytes, int64_t n_bytes,
                              const int64_t* d_text_offsets, int64_t n_texts, int32_t* d_out_ids,
                              int64_t out_capacity, int64_t* d_out_chunk_offsets, int64_t chunk_capacity,
                              int64_t* n_ids, int64_t* n_chunks, float* kernel_ms);

/* Takes the buffers of the last result out of the handle instead of copying them (no counterpart in the reference): the
 * pointers of gtk_result_view then stay valid until gtk_result_release, whatever the handle does meanwhile, also when it is
 * destroyed first; the release hands the page-locked memory back for later results.  NULL when there is nothing to take
 * -- small results and those of gtk_encode_cpu live in memory of the handle's own -- or when four results or 1 GiB are
 * out already: the caller copies then.  May be called from any thread. */
typedef struct gtk_taken gtk_taken;
GTK_API gtk_taken* gtk_result_take(gtk_tokenizer* h);
GTK_API void gtk_result_release(gtk_taken* result);

/* Device time of the stages of the last GPU encode, in milliseconds:
 * [0] chunker, [1] merge kernel, [2] output scans, [3] pack, [4] whole pipeline.
 * Also the number of kernels launched by that call (for launch accounting).
 * [4] is always measured (it is the kernel_ms the encode entry points return, the reference's one event pair,
 * gputok_binding.cu:790-805): by the kernels' own clock in GTK_MODE_OPT, by an event pair in the other modes, and as the
 * sum of the stages for batches that the host path cuts into pieces or slices (their gaps are the link's).  Host batches
 * whose chunk table the host makes itself (GTK_MODE_OPT below 6 MiB) have no chunker; where the last kernel writes the
 * results to page-locked memory that is part of its time.  [0]..[3] are measured for batches in pieces or slices, and for
 * batches that run in one piece only after gtk_set_stage_timing(h, 1); otherwise they are 0.  The events between
 * the stages cost a call of a few hundred KiB to a few MiB about a tenth of its time, which is why they are off
 * by default. */
GTK_API int gtk_last_stage_ms(const gtk_tokenizer* h, float stage_ms[5], int32_t* kernel_launches);
GTK_API int gtk_set_stage_timing(gtk_tokenizer* h, int per_stage);

/* ids -> bytes (inverse of the byte encoder + merges); the token-string writer
 * of gputok_blockbpe.cu:841-865 builds on this.  *n_out receives the byte count. */
GTK_API int gtk_decode(const gtk_tokenizer* h, const int32_t* ids, int64_t n_ids, uint8_t* out,
                       int64_t out_capacity, int64_t* n_out);

/* The symbol string the reference prints for a token (id_to_token,
 * gputok_blockbpe.cu:857).  Returns the length, -1 for an unknown id. */
GTK_API int32_t gtk_token_symbols(const gtk_tokenizer* h, int32_t id, char* buf, int32_t capacity);

/* Run all later GPU work of this handle on the caller's CUDA stream (a cudaStream_t passed as
 * void*).  NULL restores the handle's own stream, which is created non-blocking: work on it is NOT
 * ordered against the legacy default stream.  To run on the legacy default stream itself -- the
 * stream the reference always uses (gputok_binding.cu:794-799) and the one a framework reports as
 * handle 0 -- pass cudaStreamLegacy, i.e. (void*)0x1; cudaStreamPerThread is (void*)0x2.
 * Ordering contract of the device-pointer entry points (gtk_encode_device,
 * gtk_encode_chunks_noalloc): the kernels read d_bytes / offsets and write the outputs on the
 * handle's current stream; whatever produces the inputs or reuses the outputs must be ordered
 * against that stream (same stream, an event, or a synchronisation before the call).  The entry
 * points stay synchronous on return. */
GTK_API int gtk_set_stream(gtk_tokenizer* h, void* cuda_stream);

/* Threads per CTA of the one-CTA-per-chunk kernel (GTK_MODE_BASE).  Replaces the reference's compile-time
 * BLOCK_SIZE (gputok_blockbpe.cu:313-315, swept by profile_blockbpe_block_sizes.sh:9,22-25 over 128..1024):
 * 0 (default) = 64 threads for chunks up to 1 KiB, 128 up to 2 KiB, 256 beyond; 64 / 128 / 256 / 512 / 1024 = that many whatever
 * the chunk size; anything else is GTK_ERR_INVALID_ARG.  Results never depend on it. */
GTK_API int gtk_set_base_block_size(gtk_tokenizer* h, int threads);

/* Id space of the ids returned by the GPU encode entry points (no counterpart in the reference,
 * whose ids 0..255 are the byte values -- a permutation of GPT-2's own ids for the byte tokens,
 * e.g. the space byte is 32 here and 220 in GPT-2's vocab.json; ids >= 256 coincide).
 *   GTK_IDS_REFERENCE (default)  ids as the reference produces them
 *   GTK_IDS_GPT2                 ids < 256 are remapped to their position in GPT-2's byte-symbol
 *                                order, so the ids can be fed to a GPT-2 model directly
 * gtk_decode / gtk_write_token_strings expect GTK_IDS_REFERENCE ids. */
enum { GTK_IDS_REFERENCE = 0, GTK_IDS_GPT2 = 1 };
GTK_API int gtk_set_id_space(gtk_tokenizer* h, int id_space);

/* Replaces the token-string writer of the standalone binary (gputok_blockbpe.cu:841-865): writes
 * the chunks' tokens as GPT-2 symbol strings, separated by one space, one chunk per line -- the
 * format of the reference's data/output/gpu_tokens_blockbpe.txt.  chunk_id_offsets[n_chunks+1]
 * delimits the chunks inside ids (as returned by gtk_result_view). */
GTK_API int gtk_write_token_strings(const gtk_tokenizer* h, const char* path, const int32_t* ids,
                                    const int64_t* chunk_id_offsets, int64_t n_chunks);

/* Longest chunk, in bytes, that gtk_encode_chunks_noalloc accepts. */
#define GTK_NOALLOC_MAX_CHUNK_BYTES 16384

/* No counterpart in the reference (which allocates five device buffers inside every call).
 *
 * For callers that must not allocate while they tokenise: code running inside a serving loop
 * with a frozen memory budget, under a framework whose caching allocator owns all of HBM, or
 * anywhere a cudaMalloc -- which synchronises the whole device -- would stall other streams.
 * Once the handle exists this call performs no cudaMalloc/cudaFree and calls no allocating
 * library routine: the one-CTA-per-chunk greedy kernel runs with its work queue and status words
 * in a fixed array that is part of the library image; chunks that hold a segment of several
 * hundred bytes follow in a second kernel whose workspace is that array
 * (8 MiB + 256 B of device memory on every GPU that loads the library, held until the
 * process exits).
 *
 *   d_bytes[n_bytes]              text on the handle's device
 *   d_chunk_offsets[n_chunks+1]   int64, on the device: chunk c is bytes[off[c] .. off[c+1]);
 *                                 non-decreasing, 0 <= off[c] <= n_bytes.  A chunk that breaks this is
 *                                 not touched (its count is 0) and the call returns GTK_ERR_INVALID_ARG
 *   max_chunk_bytes               the caller's bound on off[c+1]-off[c]; values above
 *                                 GTK_NOALLOC_MAX_CHUNK_BYTES are rejected with GTK_ERR_CAPACITY
 *                                 before anything is launched; a chunk that breaks the bound is
 *                                 reported as GTK_ERR_CAPACITY after the kernel (its count is 0)
 *   d_out_ids[n_bytes]            int32; the ids of chunk c start at d_out_ids[off[c]] (the layout
 *                                 of the reference kernel's d_tokens_out, gputok_blockbpe.cu:530-537)
 *   d_out_counts[n_chunks]        int32 ids produced per chunk
 * The ids follow gtk_set_id_space like those of the other GPU entry points.
 *
 * The first call on a device looks up the device address of the fixed array
 * (cudaGetSymbolAddress); make that first call before any stream capture.  All calls on a
 * device share the array, which keeps the previous call's contents: the queue and status words
 * are cleared at the start of every call, the workspace is fully rewritten per chunk.  Two calls
 * that overlap on the same GPU (different handles or streams) race on it -- serialise them.
 * Synchronous on return. */
GTK_API int gtk_encode_chunks_noalloc(gtk_tokenizer* h, const uint8_t* d_bytes, int64_t n_bytes,
                                      const int64_t* d_chunk_offsets, int64_t n_chunks, int32_t max_chunk_bytes,
                                      int32_t* d_out_ids, int32_t* d_out_counts);

/* ---------------------------------------------------------------------------------------------------------------
 * Where a model takes ids in and gives them out (no counterpart in the reference, which hands its ids to a
 * framework's model, compare_generation_quality.py:418-459).
 *
 * Four operators on device memory, beside gtk_encode_device whose ids they read and gtk_decode which prints the ids
 * they find.  What they share:
 *   - ids are int32 and count rows of the table (columns of the logits) as they are: 0 .. vocab-1 in whichever id
 *     space the model was trained in (see gtk_set_id_space).  A negative id is no token (padding).  An id >= vocab is
 *     a mistake: it never touches memory and shows as NaN;
 *   - element types are GTK_F32, GTK_BF16 and GTK_F16; everything is summed in 32-bit floats and rounded once, to
 *     nearest, where it is stored;
 *   - strides count elements between the starts of neighbouring rows.  An input's may be anything >= 0 (0: every row is
 *     the same one), an output's must be >= the row's length; what lies between an output's rows is left alone.
 *     Pointers must be aligned to their elements, no more; rows that start on multiples of 16 bytes are fastest;
 *   - arrays may be read in whole pieces of 16 bytes, aligned to 16: up to 15 bytes in front of an input's first element and behind
 *     its last one, in the same 16 bytes as that.  Nothing is made of them, and nothing outside the outputs is written;
 *   - an output overlaps no input and no other output, unless it is said below that it may;
 *   - they are queued on the handle's stream (gtk_set_stream) and return without waiting, allocate nothing and may be
 *     captured into a CUDA graph (select the stream before the capture begins).  Only arguments that the host can see
 *     are reported; they are looked at before anything else, on host-only handles too.  The calling thread's current
 *     device is left as it was;
 *   - results do not depend on the run, the stream or what else the GPU does: no sum is formed in the order in which
 *     atomics arrive.
 * ------------------------------------------------------------------------------------------------------------- */
enum { GTK_F32 = 0, GTK_BF16 = 1, GTK_F16 = 2 };

/* out[i][0..dim) = scale * table[ids[i]][0..dim), i < n_ids.  A negative id gives a row of zeros, an id >= vocab a row of
 * NaN.  d_table is vocab rows of dim elements.  n_ids and vocab < 2^31, dim <= 2^20. */
GTK_API int gtk_embed(gtk_tokenizer* h, const int32_t* d_ids, int64_t n_ids, const void* d_table, int table_type,
                      int64_t vocab, int64_t dim, int64_t table_stride, float scale, void* d_out, int out_type,
                      int64_t out_stride);

/* Device memory that gtk_embed_grad needs for a call of this size (host arithmetic only). */
GTK_API int gtk_embed_grad_workspace(gtk_tokenizer* h, int64_t n_ids, int64_t vocab, int64_t dim,
                                     size_t* workspace_bytes);

/* The table's gradient: grad_table[v][0..dim) = (accumulate ? grad_table[v] : 0) + scale * the sum of grad_out[i] over
 * the i with ids[i] == v, formed in an order that is the same for the same ids.  accumulate == 0 writes every row (zeros
 * where no id points), accumulate != 0 reads and writes only rows that an id points to: the micro-batches of a step,
 * or a table whose gradient the model's last layer has written already.  Negative ids and ids >= vocab take no part.
 * d_workspace: workspace_bytes of device memory, aligned to 16 bytes, at least what gtk_embed_grad_workspace says for
 * the same sizes; its contents mean nothing before and after.  Calls (and replayed graphs) that may run at the same
 * time need workspaces of their own.  d_grad_table must not overlap d_grad_out. */
GTK_API int gtk_embed_grad(gtk_tokenizer* h, const int32_t* d_ids, int64_t n_ids, const void* d_grad_out, int out_type,
                           int64_t out_stride, float scale, int64_t vocab, int64_t dim, void* d_grad_table,
                           int table_type, int64_t table_stride, int accumulate, void* d_workspace,
                           size_t workspace_bytes);

/* Highest number of alternatives per row that gtk_token_logprobs gives. */
#define GTK_MAX_TOP 32

/* Row r of d_logits (vocab elements) stands for the distribution p_j = exp(scale * x_j - lse), lse = log sum_j
 * exp(scale * x_j); scale, above 0 and at most 1e38, is the inverse temperature.  Outputs, 32-bit floats, NULL for those that are not wanted
 * (d_targets may be NULL when d_logprob is):
 *   d_logprob[r]             log p of d_targets[r]; 0 where that is negative, NaN where it is >= vocab
 *   d_entropy[r]             -sum_j p_j log p_j
 *   d_lse[r]                 lse
 *   d_top_ids[r][0..top_k)   the top_k columns of the highest logits, highest first, of equal ones the lowest column
 *                            first (int32, rows back to back), and
 *   d_top_logprobs[r][..]    their log p.  Columns at -inf are no alternatives: places that remain hold -1 and -inf
 * A row of nothing but -inf (every id masked) has lse -inf, log p -inf, entropy 0 and no alternatives.  A row that holds
 * a NaN or +inf has NaN everywhere (a negative target's 0 excepted) and no alternatives.  Differences between a row's
 * logits that no 32-bit float holds count as infinite.  n_rows < 2^31, vocab <= 2^30, 0 <= top_k <= GTK_MAX_TOP. */
GTK_API int gtk_token_logprobs(gtk_tokenizer* h, const void* d_logits, int type, int64_t n_rows, int64_t vocab,
                               int64_t stride, float scale, const int32_t* d_targets, int top_k, float* d_logprob,
                               float* d_entropy, float* d_lse, int32_t* d_top_ids, float* d_top_logprobs);

/* The gradient of sum_r grad_logprob[r] * logprob[r] + grad_entropy[r] * entropy[r] with respect to the logits:
 *   grad_logits[r][j] = scale * (g * ([j == t] - p_j) - e * p_j * (log p_j + entropy[r]))
 * d_lse and d_entropy are what gtk_token_logprobs has given for the same logits and scale.  p_j is formed from d_lse, whose 32
 * bits are off by up to 2^-24 of itself, and p_j by as much of p_j; rows whose d_lse is 256 or more in size (logits with a large common
 * part, a mask of the type's lowest value in every column) have their sum formed again, to the precision of
 * gtk_token_logprobs, by a second reading.  d_grad_entropy may be NULL
 * (then d_entropy is not read), and so may d_grad_logprob (then d_targets is not read).  A row whose target is negative
 * or >= vocab has g = 0; rows with g = 0 and e = 0, and rows of nothing but -inf, get zeros whatever they hold.
 * d_grad_logits has the type of the logits and may be d_logits itself with the same stride; no other overlap. */
GTK_API int gtk_token_logprobs_grad(gtk_tokenizer* h, const void* d_logits, int type, int64_t n_rows, int64_t vocab,
                                    int64_t stride, float scale, const int32_t* d_targets, const float* d_lse,
                                    const float* d_entropy, const float* d_grad_logprob, const float* d_grad_entropy,
                                    void* d_grad_logits, int64_t grad_stride);

/* ---------------------------------------------------------------------------------------------------------------
 * A step of generation around a model: where requests' tokens lie in a cache of blocks, and which ids come next (no
 * counterpart in the reference, compare_generation_quality.py:418-459 leaves both to a framework).  What is said above
 * of the operators on a model's arrays holds for these three as well.
 * ------------------------------------------------------------------------------------------------------------- */

/* Largest vocabulary that gtk_sample takes. */
#define GTK_MAX_SAMPLE_VOCAB (1 << 20)

/* Draws an id from every row of d_logits (vocab elements).  With m the row's highest logit, T its temperature and the
 * columns ranked by logit, of equal ones the lower first:
 *   the first d_top_k[r] columns stay (<= 0, or as many as there are: all); logits of -inf never do;
 *   of these the fewest first ones whose weights exp((x_j - m) / T) reach d_top_p[r] of their sum (>= 1: all, <= 0: one);
 *   of these the ones with exp((x_j - m) / T) >= d_min_p[r] (<= 0: all, > 1: as 1);
 * and d_ids[r] is the lowest column at which the sum of the weights that are left, taken in the order of columns, exceeds
 * d_uniform[r] times their whole sum.  d_logprob[r] is the logarithm of the drawn column's weight over that sum.  Any of
 * d_temperature (then 1), d_top_k, d_top_p, d_min_p (then all) and d_logprob may be NULL.  Which columns stay and which one is
 * drawn is decided as in 64-bit arithmetic, and does not depend on the run.
 *   T == 0              the highest logit, of equal ones the lowest column, with log probability 0
 *   d_uniform[r] < 0    no request: id -1, log probability 0, whatever the row holds (its memory may be read)
 *   d_uniform[r] >= 1   the last column that is left with a weight above 0 in 64 bits
 *   a row of -inf       id -1, log probability -inf
 *   a row with a NaN or +inf, a NaN limit or random number, a negative, infinite or NaN temperature: id -1, log probability NaN
 * n_rows < 2^31, vocab <= GTK_MAX_SAMPLE_VOCAB. */
GTK_API int gtk_sample(gtk_tokenizer* h, const void* d_logits, int type, int64_t n_rows, int64_t vocab, int64_t stride,
                       const double* d_uniform, const float* d_temperature, const int32_t* d_top_k, const float* d_top_p,
                       const float* d_min_p, int32_t* d_ids, float* d_logprob);

/* A step of n_requests requests that have d_old_lengths[r] tokens in a cache of blocks of block_tokens tokens and will have
 * d_new_lengths[r].  Row r of d_tables holds the request's blocks, token j's in column j / block_tokens; columns behind its
 * blocks mean nothing.  Rows that grow take the blocks they lack, those that shrink (to 0: the request is over) give back
 * what they no longer need and keep the entries as they were.  A negative length is no request: its row is left alone.
 * Free blocks wait in d_queue, a ring of queue_capacity places: d_state[0] blocks have been taken from it so far, d_state[1]
 * given to it, the next one to take is at place d_state[0] % queue_capacity, the next one given goes to place d_state[1] %
 * queue_capacity.  Requests take and give in their order, and each in the order of columns; what is given back in a
 * step cannot be taken in the same.  d_state_out (int64[3]) receives both counts after the step and its status; it may be
 * d_state itself, or another array, and then the step may be queued again from the same state.  Status:
 *   0     done
 *   > 0   so many blocks are missing
 *   -1    a request has, or would have, more blocks than `columns`
 *   -2    the queue cannot be: a negative count, or one that passes 64 bits, more blocks taken than given, or more in it, with
 *         those that this step gives back and without what it takes, than it has places
 * Unless it is 0 nothing is taken, given or written, but for the counts as they were.  n_requests, columns and queue_capacity
 * < 2^31, block_tokens <= 2^20. */
GTK_API int gtk_block_tables(gtk_tokenizer* h, const int32_t* d_old_lengths, const int32_t* d_new_lengths, int64_t n_requests,
                             int block_tokens, int32_t* d_tables, int64_t columns, int64_t table_stride, int32_t* d_queue,
                             int64_t queue_capacity, const int64_t* d_state, int64_t* d_state_out);

/* Where the tokens that a step brings go: request r has those at positions d_old_lengths[r] .. d_new_lengths[r] - 1 (none
 * where it shrinks, or a length is negative), and they lie one request behind the other, as in the ids of a batch:
 *   d_offsets[r]      where request r's begin (int64[n_requests + 1], the last is the number of all)
 *   d_slots[i]        table entry * block_tokens + position % block_tokens (int64); -1 where the entry is negative or
 *                     the position is beyond `columns`
 *   d_positions[i]    the token's position, d_requests[i] its request (both may be NULL)
 * for i < capacity; places from d_offsets[n_requests] on get -1 in all three, tokens beyond capacity are left out.  d_state
 * may be NULL, or gtk_block_tables' d_state_out: after a step that was not done (a status other than 0) no request has
 * tokens here, so that nothing goes to blocks that it does not hold.  n_requests, columns and capacity < 2^31. */
GTK_API int gtk_slot_map(gtk_tokenizer* h, const int32_t* d_old_lengths, const int32_t* d_new_lengths, int64_t n_requests,
                         int block_tokens, const int32_t* d_tables, int64_t columns, int64_t table_stride, const int64_t* d_state,
                         int64_t capacity, int64_t* d_slots, int32_t* d_positions, int32_t* d_requests, int64_t* d_offsets);

/* Page-locked host memory for inputs (cudaHostAlloc / cudaFreeHost). */
GTK_API void* gtk_pinned_alloc(size_t bytes);
GTK_API void  gtk_pinned_free(void* p);

#ifdef __cplusplus
}
#endif
#endif /* GPUTOK_B200_H */
