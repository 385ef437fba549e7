/*
 * fklhip.h -- C ABI of libfklhip.so, the MI355X (gfx950) backend of the fused data-parallel path.
 *
 * This is the whole boundary between host code (plain C++20 headers under include/fused_kernel/, or any
 * language with a C FFI) and the HIP runtime + hand-written kernels.  Plain pointers and sizes only; no C++
 * types, no HIP types, no exceptions.  Every function returns 0 on success, a hipError_t value (1..9999) when
 * the HIP runtime reported an error, or one of the FKLHIP_E* codes below.  Functions are thread safe; none of
 * them synchronises the device unless its name says so.
 *
 * The reference library has no FFI: its device boundary is the CUDA runtime called from templates.  Each
 * declaration names the reference call site it stands in for (paths relative to the reference root,
 * FK/ = include/fused_kernel/).
 */
#ifndef FKLHIP_H
#define FKLHIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FKLHIP_ABI_VERSION 1

enum {
    FKLHIP_OK = 0,
    FKLHIP_EUNKNOWN_SIGNATURE = 10001, /* no kernel was built for this chain signature */
    FKLHIP_EBLOB_SIZE = 10002,         /* parameter block size does not match the signature, or exceeds FKLHIP_MAX_BLOB_BYTES */
    FKLHIP_EINVAL = 10003              /* null pointer / malformed argument */
};

enum { FKLHIP_COPY_H2H = 0, FKLHIP_COPY_H2D = 1, FKLHIP_COPY_D2H = 2, FKLHIP_COPY_D2D = 3 };

/* Largest parameter block a launch accepts.  A chain's parameters travel as by-value kernel arguments, like the
 * reference's __grid_constant__ arguments (FK/core/execution_model/executor_details/executor_kernels.h:26-30), and
 * grow with the batch (FK/core/execution_model/operation_model/batch_operations.h:164-219: one entry per plane).
 * Measured on an MI355X with ROCm 7.2: the HIP runtime accepts 1 048 584 bytes of kernel arguments and the kernel reads
 * them correctly; with 4 MiB the launch call crashes inside the runtime.  The library therefore refuses anything above
 * 1 MiB less 64 bytes (room for its own trailing arguments) with FKLHIP_EBLOB_SIZE instead of passing it on. */
#define FKLHIP_MAX_BLOB_BYTES 1048512

/* Library identity: FKLHIP_ABI_VERSION the library was built with. */
int fklhip_abi_version(void);

/* Human readable text for any code the library returns (hipGetErrorString for runtime codes).
 * Replaces cudaGetErrorString inside gpuErrchk: FK/core/utils/utils.h:100-114. */
const char *fklhip_error_string(int code);

/* Device selection.  Replaces cudaGetDevice/cudaSetDevice around allocations: FK/core/data/ptr_nd.h:154-166. */
int fklhip_get_device(int *device);
int fklhip_set_device(int device);
int fklhip_device_count(int *count);

/* Streams (always default priority).  Replaces cudaStreamCreate/Destroy/Synchronize in Stream_<GPU_NVIDIA>:
 * FK/core/execution_model/stream.h:52-109. */
int fklhip_stream_create(void **stream);
int fklhip_stream_destroy(void *stream);
int fklhip_stream_sync(void *stream);
/* 1 while a graph is being captured from the stream, else 0: nothing may be allocated for a call then. */
int fklhip_stream_is_capturing(void *stream, int *capturing);

/* Memory.  Replaces cudaMalloc / cudaMallocPitch / cudaFree / cudaMallocHost / cudaFreeHost in PtrImpl and Ptr:
 * FK/core/data/ptr_nd.h:47-126,154-250. */
int fklhip_malloc(void **ptr, size_t bytes);
int fklhip_malloc_pitch(void **ptr, size_t *pitch, size_t width_bytes, size_t height);
int fklhip_free(void *ptr);
int fklhip_host_alloc(void **ptr, size_t bytes);   /* pinned */
int fklhip_host_free(void *ptr);

/* Asynchronous copies on a stream.  Replaces cudaMemcpyAsync / cudaMemcpy2DAsync in Ptr::copy:
 * FK/core/data/ptr_nd.h:253-269. */
int fklhip_memcpy_async(void *dst, const void *src, size_t bytes, int kind, void *stream);
int fklhip_memcpy2d_async(void *dst, size_t dst_pitch, const void *src, size_t src_pitch, size_t width_bytes,
                          size_t height, int kind, void *stream);
int fklhip_memset_async(void *dst, int value, size_t bytes, void *stream);

/* Events for timing.  Replaces the cudaEvent pairs of the reference benchmarks:
 * benchmarks/fkBenchmarksCommon.h:78-132. */
int fklhip_event_create(void **event);
int fklhip_event_destroy(void *event);
int fklhip_event_record(void *event, void *stream);
int fklhip_event_sync(void *event);
int fklhip_event_elapsed_ms(float *ms, void *start, void *stop);

/*
 * Launch one fused chain.  Replaces launchTransformDPP_Kernel<<<grid, block, 0, stream>>>(details, iOps...)
 * followed by gpuErrchk(cudaGetLastError()): FK/core/execution_model/executors.h:316-351.
 *
 *   signature   the chain's type, spelled as the device-side C++ type expression (for example
 *               "Chain<Read2D<f32>,OpList<Add<f32,f32,f32>>,Write2D<f32>>"); it selects the kernel.
 *   blob        the chain's parameter block (active grid, read, compute and write parameters), laid out as the
 *               device type <signature>::Params; it is copied before the call returns, like by-value kernel
 *               arguments, so the caller may free it immediately.
 *   stream      a stream from fklhip_stream_create, or NULL for the default stream.
 *
 * fklhip_lookup resolves a signature once; the handle stays valid for the life of the process.
 */
int fklhip_lookup(const char *signature, const void **handle);
int fklhip_launch_handle(const void *handle, const void *blob, size_t blob_bytes, void *stream);
int fklhip_launch(const char *signature, const void *blob, size_t blob_bytes, void *stream);

/* A signature that was not compiled ahead of time is compiled when fklhip_lookup / fklhip_launch first see it
 * (device headers are embedded in the library; about a second per new signature, once per process; switched off by
 * the environment variable FKLHIP_JIT=0).  This is the library's stand-in for nvcc compiling the user's translation
 * unit, FK/core/execution_model/executors.h:316-351 being instantiated for whatever chain the user wrote.  When the
 * lookup fails, fklhip_jit_log returns the device compiler's messages for the last attempt on this thread (valid
 * until the next lookup on the thread).  With the environment variable FKLHIP_JIT_CACHE naming an existing directory,
 * compiled code objects are kept there (file name = hash of signature, architecture, flags and header text) and
 * reused by later processes; after such a reuse the log reads "loaded from <file>". */
int fklhip_jit_log(const char **log);

/* The bilinear kernel has two forms that give identical results: tiles, and for outputs up to 256 pixels wide whole
 * rows ("strip").  fklhip_strip_form(0) makes every later launch of the process take the tile form, fklhip_strip_form(1)
 * restores the choice by shape, a negative argument changes nothing; the return value is the previous setting (0 or 1).
 * The initial setting is 1 unless the environment variable FKLHIP_STRIP is "0" when the library first needs it.  No
 * counterpart in the reference; it exists so that tests can compare the two forms in one process. */
int fklhip_strip_form(int enable);

/* Introspection for tests and benchmarks: what the last fklhip_launch* on this thread launched.
 * kernel receives "rows", "gather" or "strip", each with "_jit" behind it for chains compiled at run time, or "rows_unaligned": the
 * kernel for rows that do not all start on dword boundaries, of the chains compiled ahead of time that have one of its own for
 * them (padding, deinterlacing, planar and circular reads; the others have one kernel for rows at every alignment).
 * The operators around a key-value cache are "heads" (norms, rotations and writes), "kv_read" and "tree_attention_TxW", with T tiles
 * of 16 rows and W waves to a workgroup; their lds_bytes are 0, as they ask for none at run time.
 * grid/block receive 3 values each. */
int fklhip_last_launch(const char **kernel, unsigned grid[3], unsigned block[3], unsigned *lds_bytes);
/* The same launch's kernel by its own name, which fklhip_last_launch gives by the form it took the place of: "rows", "flat" (planes whose rows
 * follow each other without gaps, taken as one row), "tiles", "strip", "strip_lines" (strips whose stores begin at line boundaries) or
 * "divergent", ahead of time and compiled at run time alike; "" before the first launch. */
int fklhip_last_form(const char **form);

/*
 * Attention over a quantised key-value cache: the operators a language model's server runs for new or drafted tokens.
 * The reference has them as cooperative kernels of its own beside the fused path (FK/algorithms/attention/: attention,
 * split decoding, int8 and fp8 cache reads); here they are the kernels behind the five entry points below.
 *
 * All pointers are device pointers, all strides count elements, the last dimension of rows is contiguous. 16-bit rows
 * start at multiples of 16 bytes (head_dim is a multiple of 8; their strides have to be multiples of 8). Rows of an output
 * may not overlap each other. The calls are asynchronous on `stream`, allocate nothing, record no memset and may be captured
 * into a graph. A call that returns FKLHIP_EINVAL has launched nothing; fklhip_argument_error says what was wrong. What only
 * the device can see (slots, pages, lengths, positions) is held inside its bounds by the kernels, as described at each entry.
 */
enum { FKLHIP_BF16 = 0, FKLHIP_F16 = 1 };
enum { FKLHIP_CODES_INT8 = 0, FKLHIP_CODES_E4M3 = 1 };

/* A paged cache. A cached value is code * scale with one float32 scale per token and head; codes are int8 (-127..127) or
 * e4m3 (finite, no infinities). Slot s is token s % page_tokens of page s / page_tokens.
 *   k        [pages][kv_heads][page_tokens][head_dim]          one byte each
 *   v        [pages][kv_heads][page_tokens / 4][head_dim][4]   four consecutive tokens' bytes of one element side by side
 *   k_scale  [pages][kv_heads][page_tokens], v_scale the same
 * page_tokens is 16, 32, 64, 128 or 256; k and v start at multiples of 16 bytes, the scales too. */
typedef struct fklhip_kv_cache {
    void *k, *v;
    float *k_scale, *v_scale;
    int64_t pages;
    int32_t kv_heads, page_tokens, head_dim, codes;
} fklhip_kv_cache;

/* Rows [token][head][element] of a 16-bit type. */
typedef struct fklhip_rows {
    void *data;
    int64_t token_stride, head_stride;
} fklhip_rows;

/* Query, key (and value) heads of `tokens` tokens on their way to attention. */
typedef struct fklhip_heads {
    fklhip_rows q, k, v;               /* v is read by fklhip_qkv_to_cache only */
    fklhip_rows q_out, k_out;          /* k_out is written by fklhip_qk_norm_rope only; outputs may be the inputs */
    const void *q_weight, *k_weight;   /* [head_dim] of the rows' type; NULL: no norm */
    const float *cos, *sin;            /* [positions][rot_dim / 2], rows tight; NULL with rot_dim 0 */
    const int32_t *positions;          /* [tokens]; outside of the table: the token's rotated elements are NaN */
    const int32_t *slots;              /* [tokens], fklhip_qkv_to_cache only; outside of the cache: the token is not stored */
    int64_t tokens, table_rows;
    int32_t q_heads, kv_heads, head_dim, rot_dim;
    int32_t pairs;                     /* 0: element i turns with i + rot_dim / 2, 1: 2i with 2i + 1 */
    int32_t type;
    float eps;
} fklhip_heads;

/* RMS norm of each query and key head (x * rsqrt(mean(x^2) + eps) * weight) and rotation of its first rot_dim elements by
 * the token's position ((a, b) -> (a cos - b sin, b cos + a sin)), in 32 bits, rounded once. head_dim: a multiple of 8 up
 * to 256, rot_dim: a multiple of 8 up to head_dim. */
int fklhip_qk_norm_rope(const fklhip_heads *heads, void *stream);

/* The same, with the keys (in 32 bits) and the values quantised into the cache in the same launch instead of written out. */
int fklhip_qkv_to_cache(const fklhip_heads *heads, const fklhip_kv_cache *cache, void *stream);

/* Quantises rows into the cache: scale = max |x| / 127 (448 for e4m3), code = x / scale rounded to the nearest, ties to
 * even. A row of zeros has scale 0; a row with an infinity or a NaN is stored as NaN (scale NaN, codes 0). Tokens whose
 * slot is outside of the cache (a negative one, say) are skipped. No two tokens of a call may have the same slot. */
int fklhip_kv_write(const fklhip_kv_cache *cache, const fklhip_rows *k, const fklhip_rows *v, const int32_t *slots,
                    int64_t tokens, int type, void *stream);

/* Reads `tokens` slots back as 16-bit rows; a slot outside of the cache gives zeros. */
int fklhip_kv_read(const fklhip_kv_cache *cache, const int32_t *slots, int64_t tokens, const fklhip_rows *k,
                   const fklhip_rows *v, int type, void *stream);

/* Attention of new tokens over the cache. Sequence b has context[b] cached tokens and behind them, in the cache too, its
 * q_start[b + 1] - q_start[b] new ones, whose queries are rows q_start[b].. of q. Token j of the sequence is in slot
 * page_table[b * page_table_stride + j / page_tokens] * page_tokens + j % page_tokens. Query row r sees the whole context
 * and new token u if bit u % 64 of mask[r * mask_words + u / 64] is set; without a mask, new token t sees 0..t. Query
 * heads are shared out to the key heads in order (q_heads a multiple of kv_heads). A row that sees nothing gives zeros and
 * lse -inf; a row that sees a key, and whose query holds an infinity or a NaN, gives NaN. Lengths above max_new and max_context, and tokens beyond the page table's row, are cut off; pages outside of
 * the cache are read as its last. Rows of q that are of no sequence (in front of q_start[0], cut off by max_new, at and behind
 * q_start[batch]) are zeros with lse -inf as well; q_start has to rise. With tokens, batch or max_new 0 there is no row of a
 * sequence: such a call launches nothing and leaves out and lse as they are. head_dim: 64, 96, 128, 192 or 256. */
typedef struct fklhip_attention {
    fklhip_rows q, out;
    float *lse;                        /* [tokens][q_heads] log of the sum of exponentials, or NULL */
    const int32_t *page_table, *context, *q_start;
    const uint64_t *mask;              /* [tokens][mask_words] or NULL */
    void *workspace;                   /* fklhip_tree_attention_workspace bytes; not kept between calls */
    uint64_t workspace_bytes;
    int64_t tokens, page_table_stride; /* page_table_stride: entries of a sequence's row, all of them readable */
    int32_t batch, max_new, max_context, mask_words;
    int32_t q_heads, type;
    float scale;                       /* of the scores; usually 1 / sqrt(head_dim) */
} fklhip_attention;

int fklhip_tree_attention_workspace(const fklhip_attention *call, const fklhip_kv_cache *cache, uint64_t *bytes);
int fklhip_tree_attention(const fklhip_attention *call, const fklhip_kv_cache *cache, void *stream);

/* What the last of the calls above that returned FKLHIP_EINVAL on this thread found wrong; "" before the first. */
int fklhip_argument_error(const char **text);

/* Number of chain signatures compiled into the library and the i-th of them with its parameter block size. */
int fklhip_signature_count(int *count);
int fklhip_signature_at(int index, const char **signature, size_t *blob_bytes);

#ifdef __cplusplus
}
#endif
#endif
