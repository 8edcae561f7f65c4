/*
 * browservec_hip.h -- C ABI of libbrowservec_hip.so, the MI355X (gfx950)
 * implementation of BrowserVec's data-parallel search path.
 *
 * The ABI mirrors the reference's index seam: the `VectorIndex` interface
 * (src/index/flat.ts:30-40) with its duck-typed extras (queryMasked,
 * queryBatch, setNprobe, getters; src/index.ts:78-80, 352-354, 477-501,
 * 702-750), the engine's `DeviceContext` (src/engine/device.ts:3-9) and
 * `BrowserVec.rerankExact` (src/index.ts:583-594).  Plain pointers and sizes
 * only; every call returns a status code and leaves a message for
 * bv_last_error() on failure.  Host pointers are caller-owned and consumed
 * before the call returns.
 *
 * Scores follow the reference: higher is closer; cosine and dot are the dot
 * product (rows and queries arrive already normalized for cosine, as
 * Store.prepare does), l2 is the negative squared distance.  Results come
 * back in canonical order: score descending, then row ascending.
 *
 * Thread safety: one index may be used by one thread at a time (the
 * reference awaits queries serially per store, src/engine/profile.ts:11-14);
 * different indexes may be used concurrently.
 */
#ifndef BROWSERVEC_HIP_H
#define BROWSERVEC_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define BV_ABI_VERSION 1

/* Status codes.  The message text of BV_E_INVALID for a length mismatch is
 * the reference's: "expected <n> floats, got <m>" (src/index/flat.ts:96-98). */
#define BV_OK 0
#define BV_E_INVALID 1     /* bad argument (lengths, dims, k, null pointers)          */
#define BV_E_UNSUPPORTED 2 /* combination the reference rejects (buildIndex, index.ts:119-141) */
#define BV_E_DEVICE_LOST 3 /* "GPU device lost; re-create the store" (flat.ts:137)  */
#define BV_E_OOM 4         /* device allocation failed                             */
#define BV_E_HIP 5         /* any other HIP runtime error                          */
#define BV_E_STATE 6       /* call not valid in the current state                  */

/* Index kinds: the classes buildIndex constructs (src/index.ts:105-142). */
#define BV_KIND_FLAT 0     /* FlatIndex      src/index/flat.ts:42      */
#define BV_KIND_QUANT 1    /* QuantIndex     src/index/quant.ts:21     */
#define BV_KIND_IVF 2      /* IVFIndex       src/index/ivf.ts:51       */
#define BV_KIND_IVFQUANT 3 /* IVFQuantIndex  src/index/ivfquant.ts:33  */

/* Metric (src/types.ts `Metric`). */
#define BV_METRIC_COSINE 0
#define BV_METRIC_DOT 1
#define BV_METRIC_L2 2

/* Scorer for quantized kinds.  ASYM is the reference's (fp32 rotated query x
 * dequantized codes, src/engine/wgsl/distanceQ{8,4,1}.ts).  HAMMING (1-bit
 * only) scores P - 2*popcount(code ^ sign_bits(query)); INT8SYM (int8 only)
 * quantizes the query with quantizeRow and scores the exact int32 dot.  The
 * last two have no reference counterpart; they are integer and exact. */
#define BV_SCORER_ASYM 0
#define BV_SCORER_HAMMING 1
#define BV_SCORER_INT8SYM 2

typedef struct bv_device bv_device;
typedef struct bv_index bv_index;
typedef struct bv_graph bv_graph;

/* Index description: buildIndex's arguments (dim, metric, quantBits, quant,
 * ann, chunkRows; src/index.ts:105-113) with the QuantConfig and IVFParams
 * fields (src/types.ts:116-128, src/index/ivf.ts:29-49).  Zero means "the
 * reference default" for every optional field. */
typedef struct bv_index_desc {
    uint32_t size;          /* sizeof(bv_index_desc); 72 (no ivf_incremental) is read
                             * with ivf_incremental = 0                               */
    uint32_t kind;          /* BV_KIND_*                                             */
    uint32_t dim;           /* vector dimension (> 0)                                */
    uint32_t metric;        /* BV_METRIC_*                                           */
    uint32_t bits;          /* 0 (fp32), 8, 4, 1                                     */
    uint32_t scorer;        /* BV_SCORER_*                                           */
    uint32_t seed;          /* rotation seed; has_seed=0 -> 0x9e3779b9 (index.ts:71) */
    uint32_t has_seed;
    uint32_t rounds;        /* Hadamard rounds; 0 -> 2 (index.ts:115)                */
    uint32_t chunk_rows;    /* forced rows per chunk (reported only; one buffer here) */
    uint32_t nlist;         /* IVF: 0 -> round(sqrt(rows)) clamped [16,4096]         */
    uint32_t nprobe;        /* IVF: 0 -> tuned or 5% of nlist                        */
    uint32_t sample_size;   /* IVF reservoir; 0 -> 50000 (min 1024)                  */
    uint32_t train_size;    /* IVF k-means rows; 0 -> 16384                          */
    uint32_t iters;         /* IVF Lloyd iterations; 0 -> 8 (quant) / 8 (fp32)       */
    uint32_t ivf_seed;      /* IVF seed; has_ivf_seed=0 -> reference default         */
    uint32_t has_ivf_seed;
    float target_recall;    /* IVF: < 0 -> unset                                     */
    uint32_t ivf_incremental; /* IVF: 1 -> appends after a build assign the new rows
                               * to the current centroids and extend the lists; 0 ->
                               * the reference's rebuild on the next query
                               * (src/index/ivfquant.ts:462)                          */
} bv_index_desc;

/* Stats (the index-derived fields of `Stats`, src/types.ts:253-300, and
 * src/index.ts:702-750) plus device timings. */
typedef struct bv_index_stats {
    uint64_t rows;            /* VectorIndex.size                                     */
    uint32_t dim;
    uint32_t padded_dim;      /* quantized kinds: padToPow2(dim)                      */
    uint32_t words_per_row;   /* quantized kinds                                      */
    uint32_t bits;
    uint32_t chunk_count;     /* chunkCount getter                                    */
    uint32_t nlist;           /* nlist getter (0 until built)                         */
    uint32_t nprobe;          /* nprobe getter (0 until built)                        */
    float tuned_recall;       /* tunedRecall getter; < 0 when unset                   */
    double last_query_ms;     /* host wall time of the last query call                */
    double last_query_gpu_ms; /* device time of the last query (HIP events)           */
    double build_ms;          /* last IVF build                                       */
    uint64_t device_bytes;    /* HBM held by the index                                */
    uint64_t last_scanned_rows;
    uint64_t build_exact_rows;  /* last IVF build's final assignment: rows assigned by
                                 * the exact fp32 arithmetic alone (all of them, or
                                 * those the int8 matrix pass left open)            */
} bv_index_stats;

/* ---- errors / version ---------------------------------------------------- */
const char *bv_last_error(void); /* thread-local message of the last failure */
int bv_abi_version(void);

/* ---- device (DeviceContext, src/engine/device.ts:3-76) -------------------- */
/* acquireDevice (device.ts:22-50): open HIP device `ordinal`. */
int bv_device_open(int ordinal, bv_device **out);
/* device.destroy() (src/index.ts:753-756). */
int bv_device_close(bv_device *dev);
/* DeviceContext.lost (device.ts:68-76). */
int bv_device_is_lost(const bv_device *dev, int *lost);
/* Failure injection for tests of the error paths.  The reference's device
 * loss comes from the browser (GPUDevice.lost sets DeviceContext.lost,
 * src/engine/device.ts:68-76; queries then throw "GPU device lost; re-create
 * the store", src/index/flat.ts:137); these host-side flags force the same
 * conditions without touching the GPU. */
#define BV_INJECT_LOST 1       /* mark the device lost: every later call fails with BV_E_DEVICE_LOST */
#define BV_INJECT_APPEND_OOM 2 /* the next append fails as if a device allocation failed; the index is unchanged */
#define BV_INJECT_APPEND_LATE 3 /* the next append fails after its rows are uploaded and encoded, before its
                                 * reservoir sample and lists are committed; the index is unchanged */
#define BV_INJECT_SLOTS_OOM 4 /* the next slot scan's scratch does not fit: the query takes another path */
int bv_debug_inject(bv_device *dev, int what);
/* Device name, compute-unit count and HBM size. */
int bv_device_info(const bv_device *dev, char *name, uint32_t name_len, uint32_t *cu_count, uint64_t *hbm_bytes);

/* ---- index lifecycle ------------------------------------------------------ */
/* buildIndex (src/index.ts:105-142): same validation and error messages. */
int bv_index_create(bv_device *dev, const bv_index_desc *desc, bv_index **out);
/* VectorIndex.destroy (flat.ts:39). */
int bv_index_destroy(bv_index *idx);
/* VectorIndex.size (flat.ts:31). */
int bv_index_size(const bv_index *idx, uint64_t *rows);

/* VectorIndex.append (flat.ts:37, quant.ts:129-140, ivfquant.ts:216-233):
 * `data` holds n_floats = count*dim prepared floats (normalized for cosine).
 * Quantized kinds rotate+quantize on the device. */
int bv_index_append(bv_index *idx, const float *data, uint64_t n_floats, uint64_t count);

/* ---- queries ---------------------------------------------------------------- */
/* VectorIndex.query (flat.ts:38): top-k of one query.  Flat kinds are exact;
 * quantized kinds return the approximate top-k by code score (the caller
 * re-ranks, as BrowserVec.query does).  *n_out = min(k, rows).  Any k on
 * flat kinds (above 1024: every row's score, then a device sort); IVF
 * kinds serve k <= 1024. */
int bv_index_query(bv_index *idx, const float *q, uint32_t k, uint32_t *rows, float *scores, uint32_t *n_out);

/* queryMasked (flat.ts:128-130, quant.ts:174-176): rows whose bit (LSB-first,
 * row r -> word r>>5) is clear never enter the top-k; *n_out may be < k. */
int bv_index_query_masked(bv_index *idx, const float *q, uint32_t k, const uint32_t *mask_words,
                          uint64_t n_words, uint32_t *rows, float *scores, uint32_t *n_out);

/* queryBatch (src/index.ts:499-501): nq queries (nq*dim floats); results
 * row-major [nq][k], n_out[nq].  Equal to looping bv_index_query: rows and
 * score bits (8 or more queries on a flat fp32 or int8 / int4 index run on
 * the matrix cores as a prefilter; the rows it keeps are scored with the
 * single-query arithmetic). */
int bv_index_query_batch(bv_index *idx, const float *queries, uint32_t nq, uint32_t k, uint32_t *rows,
                         float *scores, uint32_t *n_out);

/* setNprobe (ivfquant.ts:154-156): per-query override for the next query
 * call, consumed once (0 clears). */
int bv_index_set_nprobe(bv_index *idx, uint32_t nprobe);

/* BrowserVec.rerankExact (src/index.ts:583-594): score the candidate rows
 * with Store.dotRow's f64 arithmetic (store.ts:114-130) against the stored
 * fp32 rows and return their top-k.  Needs rows kept on the device (all
 * quantized kinds keep them). */
int bv_index_rerank(bv_index *idx, const float *q, const uint32_t *cand, uint32_t n_cand, uint32_t k,
                    uint32_t *rows, float *scores, uint32_t *n_out);

/* BrowserVec.queryRowsExact (src/index.ts:445-464): the exact score of each
 * listed row against q -- Store.dotRow (store.ts:114-130), or Store.l2Row
 * (store.ts:137-160) on an l2 index, in their f64 order, stored as f32 --
 * and the top k of them, ordered (score desc, row asc).  Any k and any
 * number of rows; a row >= size fails with BV_E_INVALID.  The reference
 * runs this on the host for filters that match few rows (and for selective
 * filters on IVF indexes); here it runs on the stored device rows. */
int bv_index_query_rows(bv_index *idx, const float *q, const uint32_t *list, uint64_t n_list, uint32_t k,
                        uint32_t *rows, float *scores, uint32_t *n_out);
/* bv_index_query_rows over the rows whose bit is set in mask_words (the
 * queryMasked layout, scoreMask.ts:23-98: bit r & 31 of word r >> 5; bits at
 * or past size are ignored, a short mask leaves the remaining rows out).  The
 * row list is built on the device from the mask. */
int bv_index_query_rows_masked(bv_index *idx, const float *q, const uint32_t *mask_words, uint64_t n_words,
                               uint32_t k, uint32_t *rows, float *scores, uint32_t *n_out);

/* BrowserVec.query's quantized path in one device round trip (index.ts:
 * 402-421): approximate top-`fetch`, then exact re-rank to top-`k`.  With
 * fetch == 0 no re-rank happens and the approximate top-k is returned.
 * queries: nq*dim floats; rows/scores [nq][k]; n_out[nq]. */
int bv_index_search(bv_index *idx, const float *queries, uint32_t nq, uint32_t fetch, uint32_t k,
                    uint32_t *rows, float *scores, uint32_t *n_out);

/* ---- device-resident variants (serving loops, benchmarks) ------------------ */
/* Same as bv_index_search with every pointer in device memory; enqueued on
 * the index's stream and returns without waiting, except for batches of 8 or
 * more queries on a flat index, which may run on the matrix cores and then
 * wait once (fp32 rows: once per 1,024 queries, or fewer at a time where k
 * and the row count are large; a count per query is read back). */
int bv_index_search_device(bv_index *idx, const float *d_queries, uint32_t nq, uint32_t fetch, uint32_t k,
                           uint32_t *d_rows, float *d_scores, uint32_t *d_n_out);

/* Query streams for bv_index_search_device (no counterpart in the
 * reference; for callers that keep several single queries in flight):
 * n = 2 to 4 lets consecutive fused calls (fewer than 8 queries per call,
 * no mask) take the index's stream and n - 1 further streams in turn, each
 * with its own scan scratch (IVF indexes: also its own probe and candidate
 * buffers), so one query's final selection overlaps the next query's scan.
 * Calls in flight may then run at once: each needs its own output buffers.
 * bv_index_sync waits for every stream; appends wait for queries still
 * running.  n = 1 (default): one stream. */
int bv_index_set_query_streams(bv_index *idx, uint32_t n);
/* bv_index_search_device for callers that cannot allocate device memory
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  It has no counterpart in the reference.  Every query runs the
 * fused single-query scan with its scratch in a library-owned array of
 * BV_NOALLOC_SCRATCH_BYTES per GPU, held until the process ends; the call
 * allocates nothing and launches only kernels (no memset or copy nodes).
 * Serves flat indexes and quantized indexes whose scan transforms queries
 * in-kernel (int8 / int4 / 1-bit / Hamming at padded dimensions 64..1024),
 * not IVF.  BV_E_INVALID when nq, fetch and k need more scratch than the
 * array holds (about 10.5 MB per query at 1M rows and fetch 100).  All calls
 * on one GPU share the array: calls that overlap on that GPU (other streams,
 * other threads, other indexes) race. */
#define BV_NOALLOC_SCRATCH_BYTES (64u << 20)
int bv_index_search_device_noalloc(bv_index *idx, const float *d_queries, uint32_t nq, uint32_t fetch, uint32_t k,
                                   uint32_t *d_rows, float *d_scores, uint32_t *d_n_out);
/* Append rows that already live in device memory (count*dim floats). */
int bv_index_append_device(bv_index *idx, const float *d_data, uint64_t count);
/* Wait for all work enqueued on the index's stream. */
int bv_index_sync(bv_index *idx);
/* The index's HIP stream (hipStream_t) as an opaque pointer. */
int bv_index_stream(bv_index *idx, void **stream);
/* Per-kernel device timing with HIP events on the index's stream.  enable=1
 * starts counting (and resets), enable=0 stops.  Reports the summed duration
 * and launch count of the scan kernel (the dominant one). */
int bv_index_kernel_timing(bv_index *idx, int enable, double *scan_ms, uint64_t *scan_launches);

/* ---- stats / parity exports --------------------------------------------------- */
int bv_index_get_stats(bv_index *idx, bv_index_stats *out);
/* Codes and scales of rows [row0, row0+count) (words_per_row u32 per row). */
int bv_index_export_codes(bv_index *idx, uint64_t row0, uint64_t count, uint32_t *words, float *scales);
/* The scan's score for every row for one query (rows floats): the dense
 * scores the reference's distance kernels leave in their score buffer. */
int bv_index_export_scores(bv_index *idx, const float *q, float *scores);
/* The device-rotated query (padded_dim floats), quantized kinds only. */
int bv_index_export_rotated_query(bv_index *idx, const float *q, float *rotated);

/* ---- IVF ------------------------------------------------------------------------ */
/* IVFIndex / IVFQuantIndex build (src/index/ivf.ts:191-259,
 * src/index/ivfquant.ts:248-312): k-means on the reservoir sample, final
 * assignment, CSR lists.  Queries build on demand after appends, as the
 * reference does; this entry builds now.  With desc.ivf_incremental, appends
 * after a build extend the lists instead (the new rows assigned to the
 * current centroids); this entry then retrains over the reservoir and
 * reassigns every row, giving the lists the reference would build. */
int bv_index_build(bv_index *idx);
/* The built IVF state for parity checks: centroids (nlist x D floats, D =
 * padded_dim for quantized kinds, dim for fp32), list offsets (nlist+1) and
 * list rows (rows, ascending within a list).  Any pointer may be null.
 * Stale lists are built first, as a query would; lists extended by
 * incremental appends are exported as they stand. */
int bv_index_export_ivf(bv_index *idx, float *centroids, uint32_t *list_off, uint32_t *list_rows);

/* Index section for snapshots (src/persist/format.ts:1-22, whose v2 HNSW
 * graph section is the precedent; src/index.ts:673-700 re-encodes and
 * re-trains on load instead): the codes and scales of quantized kinds and the
 * IVF state (reservoir rows and ids, centroids, CSR lists, tuned nprobe).
 * The snapshot's fp32 rows stay where the reference keeps them.
 * bv_index_save_section writes *size bytes to buf when cap >= *size; with
 * buf == NULL or a smaller cap it only reports *size. */
int bv_index_save_section(bv_index *idx, void *buf, uint64_t cap, uint64_t *size);
/* Fills an empty index from the snapshot's rows (count*dim prepared floats,
 * as append takes them) and a saved section, without encoding or training.
 * The index must have been created with the descriptor the section was saved
 * under (BV_E_INVALID otherwise).  Appends after a load continue exactly as
 * on the saved index. */
int bv_index_load_section(bv_index *idx, const float *data, uint64_t n_floats, uint64_t count, const void *section,
                          uint64_t bytes);
/* pickProbes' scores (src/index/ivfquant.ts:495-509: the f64 4-way strided
 * dot of the rotated query with every centroid, stored as f32) for nq
 * queries: scores[nq][nlist].  Batches of 8 or more run the batched probe
 * kernel, fewer the single-query one; both give the same bits. */
int bv_index_export_probe_scores(bv_index *idx, const float *queries, uint32_t nq, float *scores);

/* ---- graph search (HNSW layer 0) ------------------------------------------ */
/* HNSWGpuSearcher (src/index/hnswGpu.ts:28-244): the host's HNSW build keeps
 * the graph; this object holds the corpus rows and the flat layer-0
 * adjacency on the device and beam-searches query batches
 * (src/engine/wgsl/graphSearch.ts:62-259), one workgroup per query.  degree is
 * the adjacency's fixed out-degree (2M), at most 64; metric BV_METRIC_* (the
 * rows and queries arrive prepared, as for an index). */
int bv_graph_create(bv_device *dev, uint32_t dim, uint32_t metric, uint32_t degree, bv_graph **out);
int bv_graph_destroy(bv_graph *g);
/* HNSWGpuSearcher.append (hnswGpu.ts:83-109): mirror appended rows. */
int bv_graph_append(bv_graph *g, const float *data, uint64_t n_floats, uint64_t count);
/* HNSWGpuSearcher.uploadGraph (hnswGpu.ts:112-126): the layer-0 adjacency,
 * rows x degree row ids, 0xffffffff for an empty slot.  Rows past the
 * adjacency have no neighbours; ids at or past the corpus rows are skipped. */
int bv_graph_upload(bv_graph *g, const uint32_t *links, uint64_t rows);
/* HNSWGpuSearcher.search (hnswGpu.ts:134-206): beam width
 * min(max(ef, k), 256), as many expansions, seeds = entry plus up to seven
 * rows spread over the adjacency; per query the beam's ids deduped, sorted
 * by score (-distance: dot for dot / cosine, -squared distance for l2) with
 * ties in beam order, the first k: rows / scores [nq][k], n_out[nq]. */
int bv_graph_search(bv_graph *g, const float *queries, uint32_t nq, uint32_t k, uint32_t ef, uint32_t entry,
                    uint32_t *rows, float *scores, uint32_t *n_out);
/* Parity export: the raw beams ([nq][256] distances and ids, unsorted, empty
 * slots 3.4e38 / 0xffffffff) for explicit seeds, beam width and expansion
 * cap. */
int bv_graph_search_beams(bv_graph *g, const float *queries, uint32_t nq, const uint32_t *entries,
                          uint32_t n_entries, uint32_t ef, uint32_t iter_cap, float *beam_dist, uint32_t *beam_id);

/* ---- an embedding model's operators ------------------------------------------ */
/* What turns text into the vectors an index holds, beside it on the GPU: the
 * reference's embedder runs in another library (src/embed/transformers.ts),
 * these are the operators such a model's forward pass is made of.  Every
 * pointer is device memory unless it says otherwise; a call checks its
 * arguments, enqueues kernels on the handle's stream and returns without
 * waiting.  Matrices and heads have contiguous last dimensions and strides in
 * elements (0: packed); every alignment and size works, 16-byte aligned rows
 * run fastest.  Sums, softmax statistics and norms are 32-bit floats; results
 * are rounded once to the output's type (in bv_embed_attention a key's weight
 * as well, to the type of q, k and v, before it multiplies its value), and the
 * same call on the same inputs gives the same bits.  Outputs may not overlap inputs except where a
 * description allows it.
 *
 * A handle is used by one thread at a time.  Its workspaces, one for each
 * stream it is used on, grow with the largest call so far and are held until
 * the handle is destroyed: after one call of a size on a stream, further calls
 * of it there allocate nothing.  Calls launch only kernels and can be captured
 * into a HIP graph.  Each capture has workspaces of its own, held until the
 * handle is destroyed, so that graphs may run beside each other and beside
 * other calls; runs of the same graph follow one another. */
#define BV_F32 0
#define BV_F16 1
#define BV_BF16 2

typedef struct bv_embed bv_embed;

/* A handle with a stream of its own (not ordered with the null stream). */
int bv_embed_create(bv_device *dev, bv_embed **out);
/* Waits for the device. */
int bv_embed_destroy(bv_embed *e);
/* Run further calls on another stream (hipStream_t; NULL is the device's
 * default stream), an index's (bv_index_stream) to append or search without
 * waiting in between.  Orders nothing: calls on two streams may run at once. */
int bv_embed_set_stream(bv_embed *e, void *stream);
int bv_embed_stream(bv_embed *e, void **stream);
int bv_embed_sync(bv_embed *e);

/* y = act(x w^T + bias) + residual: x [m][k], w [n][k] and bias [n] in dtype
 * (BV_F16 or BV_BF16), residual and y [m][n] in out_dtype (dtype or BV_F32).
 * bias and residual may be NULL; residual may be y itself. */
#define BV_ACT_NONE 0
#define BV_ACT_RELU 1
#define BV_ACT_GELU 2      /* x Phi(x)                                               */
#define BV_ACT_GELU_TANH 3 /* x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))) / 2        */
#define BV_ACT_SILU 4      /* x / (1 + exp(-x))                                      */
typedef struct bv_embed_linear_args {
    uint32_t size;        /* sizeof(bv_embed_linear_args) */
    uint32_t dtype;
    uint32_t out_dtype;
    uint32_t activation;  /* BV_ACT_* */
    uint64_t m;
    uint32_t n;
    uint32_t k;
    const void *x;
    const void *w;
    const void *bias;
    const void *residual;
    void *y;
    uint64_t x_stride;    /* elements from a row to the next; 0: packed */
    uint64_t w_stride;
    uint64_t residual_stride;
    uint64_t y_stride;
} bv_embed_linear_args;
int bv_embed_linear(bv_embed *e, const bv_embed_linear_args *args);

/* Rotary positions: the first rot_dim elements of every head turn in pairs,
 * (a, b) -> (a cos - b sin, b cos + a sin); the others are copied.  Pairs are
 * elements i and i + rot_dim/2, or 2i and 2i+1 with interleaved.  table holds
 * a row per position, [table_rows][rot_dim/2] pairs (cos, sin) of 32-bit floats
 * (bv_embed_rotary_table); positions one int32 per token (NULL: 0, 1, ...).  A
 * position outside the table turns its token's elements into NaN.  q
 * [tokens][heads_q][head_dim] and k [tokens][heads_k][head_dim] in dtype; k may
 * be NULL with heads_k 0.  q_out may be q and k_out k, with the same strides. */
typedef struct bv_embed_rotary_args {
    uint32_t size;        /* sizeof(bv_embed_rotary_args) */
    uint32_t dtype;
    uint32_t heads_q;
    uint32_t heads_k;
    uint32_t head_dim;
    uint32_t rot_dim;     /* even, at most head_dim */
    uint32_t interleaved;
    uint32_t table_rows;
    uint64_t tokens;
    const float *table;
    const int32_t *positions;
    const void *q;
    const void *k;
    void *q_out;
    void *k_out;
    uint64_t q_stride;    /* elements from a token to the next; 0: packed */
    uint64_t q_head_stride;
    uint64_t k_stride;
    uint64_t k_head_stride;
    uint64_t q_out_stride;
    uint64_t q_out_head_stride;
    uint64_t k_out_stride;
    uint64_t k_out_head_stride;
} bv_embed_rotary_args;
int bv_embed_rotary(bv_embed *e, const bv_embed_rotary_args *args);

/* The table of bv_embed_rotary in host memory: cos and sin of position times
 * frequency in 64 bits, rounded to 32.  Pair i's frequency is
 * f = base^(-2i/rot_dim), scaled for contexts `factor` times the original:
 *   BV_ROTARY_NONE    f
 *   BV_ROTARY_LINEAR  f / factor
 *   BV_ROTARY_BASE    f of the base times factor^(rot_dim/(rot_dim-2))
 *   BV_ROTARY_PARTS   f (g + (1-g)/factor): g = 1 for pairs that turn at least
 *                     high_turns times over original_rows positions, 0 for
 *                     those that turn at most low_turns times, linear between
 * magnitude multiplies cos and sin (0: 1).  n_floats must be
 * table_rows * rot_dim. */
#define BV_ROTARY_NONE 0
#define BV_ROTARY_LINEAR 1
#define BV_ROTARY_BASE 2
#define BV_ROTARY_PARTS 3
typedef struct bv_embed_rotary_scaling {
    uint32_t size;        /* sizeof(bv_embed_rotary_scaling) */
    uint32_t kind;        /* BV_ROTARY_* */
    double base;
    double factor;
    double original_rows;
    double low_turns;
    double high_turns;
    double magnitude;
} bv_embed_rotary_scaling;
int bv_embed_rotary_table(const bv_embed_rotary_scaling *scaling, uint32_t table_rows, uint32_t rot_dim, float *table,
                          uint64_t n_floats);

/* o = softmax(scale q k^T) v per packed sequence and head: sequence s has the
 * queries cu_q[s] to cu_q[s+1] of q [tokens_q][heads_q][head_dim] and the keys
 * cu_k[s] to cu_k[s+1] of k, v [tokens_k][heads_k][head_dim] (dtype BV_F16 or
 * BV_BF16; head_dim at most 256; heads_q a multiple of heads_k, query head h
 * reads key head h / (heads_q/heads_k); tokens_k and tokens_q heads_q/heads_k
 * at most 2^31 - 1025).  cu_q, cu_k: batch + 1 ascending
 * int32, clipped to the tokens there are.  causal: a sequence's last query
 * sees its last key, each query before it one key less.  A query that sees no
 * key gives zeros.  Keys and values that a query does not see have no effect
 * on it, whatever they hold.  scale 0: 1/sqrt(head_dim).  max_q and max_k are
 * the longest lengths as far as the caller knows them (0: unknown); they only
 * steer how the work is split, never which of it is done.  Queries outside
 * every sequence leave their rows of o as they are. */
typedef struct bv_embed_attention_args {
    uint32_t size;        /* sizeof(bv_embed_attention_args) */
    uint32_t dtype;
    uint32_t heads_q;
    uint32_t heads_k;
    uint32_t head_dim;
    uint32_t causal;
    uint32_t batch;
    uint32_t max_q;
    uint32_t max_k;
    float scale;
    uint64_t tokens_q;
    uint64_t tokens_k;
    const void *q;
    const void *k;
    const void *v;
    void *o;
    const int32_t *cu_q;
    const int32_t *cu_k;
    uint64_t q_stride;    /* elements from a token to the next; 0: packed */
    uint64_t q_head_stride;
    uint64_t k_stride;
    uint64_t k_head_stride;
    uint64_t v_stride;
    uint64_t v_head_stride;
    uint64_t o_stride;
    uint64_t o_head_stride;
} bv_embed_attention_args;
int bv_embed_attention(bv_embed *e, const bv_embed_attention_args *args);

/* The norm of token rows and their pooling to one vector a sequence.
 * x [tokens][dim] in dtype; each row becomes
 *   BV_NORM_NONE   x
 *   BV_NORM_LAYER  (x - mean) / sqrt(var + eps)
 *   BV_NORM_RMS    x / sqrt(mean(x^2) + eps)
 * times weight plus bias ([dim] in weight_dtype, each may be NULL).  With
 * BV_POOL_NONE y holds those rows, [tokens][dim] in out_dtype (y may be x where
 * the types and strides are the same).  Otherwise y [batch][dim], out_dtype
 * BV_F32, holds per sequence cu[s] to cu[s+1] (batch + 1 ascending int32,
 * clipped to the tokens there are) their mean, the first or the last of them,
 * and with unit divided by its 2-norm: the rows bv_index_append_device and the
 * queries bv_index_search_device take.  An empty sequence gives zeros, a
 * vector of norm zero stays as it is.  Squares are 32-bit floats too: the norms
 * and the 2-norm are for elements whose squares, and their sum, are no larger
 * than 3e38, and for rows whose sum of squares is above 1e-38. */
#define BV_NORM_NONE 0
#define BV_NORM_LAYER 1
#define BV_NORM_RMS 2
#define BV_POOL_NONE 0
#define BV_POOL_MEAN 1
#define BV_POOL_FIRST 2
#define BV_POOL_LAST 3
typedef struct bv_embed_norm_args {
    uint32_t size;        /* sizeof(bv_embed_norm_args) */
    uint32_t dtype;
    uint32_t out_dtype;
    uint32_t weight_dtype;
    uint32_t norm;        /* BV_NORM_* */
    uint32_t pool;        /* BV_POOL_* */
    uint32_t unit;
    uint32_t batch;
    uint32_t dim;
    float eps;
    uint64_t tokens;
    const void *x;
    const void *weight;
    const void *bias;
    const int32_t *cu;
    void *y;
    uint64_t x_stride;    /* elements from a row to the next; 0: packed */
    uint64_t y_stride;
} bv_embed_norm_args;
int bv_embed_norm(bv_embed *e, const bv_embed_norm_args *args);

#ifdef __cplusplus
}
#endif

#endif /* BROWSERVEC_HIP_H */
