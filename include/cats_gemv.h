/*
 * cats_gemv.h -- C ABI of the gfx950 CATS sparse-MLP decode kernels.
 *
 * Every entry point takes plain device pointers, sizes and a HIP stream and returns a
 * cats_status_t.  Nothing here allocates, frees or synchronises (cats_read_count is the one
 * documented exception: it has to hand a device counter back to the host, and its first call
 * allocates one pinned host word for that).  A launch failure is reported as CATS_ERR_LAUNCH
 * from the status of that launch alone; errors left behind by the caller's earlier HIP calls are
 * neither returned nor cleared.  All launches go
 * to the stream that is passed in.  The entry points are what a `TORCH_LIBRARY(flash_gemv, m)`
 * shim, a ctypes loader or any other FFI binds; each one names the reference interface it
 * stands in for (paths relative to the CATS tree).
 *
 * Conventions
 *   B      rows of the activation matrix (batch * seq, decode => seq == 1); 1 <= B <= CATS_MAX_BATCH
 *   H      hidden size, I intermediate size
 *   dtype  cats_dtype_t; x, weights and dtype-typed outputs all share it
 *   x        (B, H)  row-major
 *   wgate    (I, H)  row-major  (nn.Linear layout: one row per neuron)
 *   wup      (I, H)  row-major
 *   wdown_t  (I, H)  row-major, "neuron-major": row j is column j of the HF down_proj.weight
 *   wdown    (H, I)  row-major  (HF nn.Linear layout)
 *   flag     (B, I)  one byte per entry, 0 or 1 (torch.bool storage)
 *   Rows must be 16-byte aligned: H * sizeof(dtype) % 16 == 0 and all base pointers 16-byte
 *   aligned (I * sizeof(dtype) % 16 == 0 as well where I is a row length: wdown, a, z).
 *
 * Activation and mask rule (experiments/models/sparse_silu/ugly_utils.py:895-899,
 * flash_gemv/flash_gemv/__init__.py:41,46):
 *   g  = round_dtype(sum_k x[b,k] * wgate[j,k])        fp32 accumulation
 *   a  = round_dtype(g / (1 + exp(-g)))                SiLU evaluated in fp32
 *   active(b,j)  <=>  |a| > round_dtype(threshold)     strict, compared on the stored value
 *   z  = active ? round_dtype(a * round_dtype(sum_k x[b,k] * wup[j,k])) : 0
 *   y  = round_dtype(sum_j z[b,j] * wdown_t[j,:])      fp32 accumulation
 * A weight row of wup / wdown_t is fetched only if some row b of the batch has it active.
 */
#ifndef CATS_GEMV_H
#define CATS_GEMV_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { CATS_F16 = 0, CATS_BF16 = 1, CATS_F32 = 2 } cats_dtype_t;

typedef enum {
  CATS_OK = 0,
  CATS_ERR_DTYPE = 1,      /* dtype is not a cats_dtype_t */
  CATS_ERR_SHAPE = 2,      /* non-positive or unsupported H / I */
  CATS_ERR_ALIGN = 3,      /* a pointer or row pitch is not 16-byte aligned */
  CATS_ERR_BATCH = 4,      /* B outside 1..CATS_MAX_BATCH */
  CATS_ERR_NULL = 5,       /* a required pointer is NULL */
  CATS_ERR_WORKSPACE = 6,  /* workspace missing or smaller than cats_workspace_bytes() */
  CATS_ERR_LAUNCH = 7,     /* the HIP runtime refused a launch; hipGetLastError() has details */
  CATS_ERR_SCRATCH = 8     /* cats_mlp_noalloc: the call does not fit the library's built-in scratch */
} cats_status_t;

#define CATS_MAX_BATCH 16  /* 1..8 rows are one pass over the weights.  9..16 rows: the whole-MLP entry points (cats_mlp, the
                            * layer-tail calls, cats_up_down, cats_mlp_rowmajor_down), cats_gate_flag, cats_gate_up and cats_up_flag
                            * (16-bit types, rows of up to 4360 elements, and 4416 or 4480 on cache lines; fp32 rows of any
                            * length in cats_mlp, cats_mlp_rowmajor_down, cats_gate_flag and cats_gate_up) and cats_down_flag (16-bit types) still
                            * read gate and up once; every other case is two passes of at most eight rows */

/* Library identification / error text.  No reference counterpart (the reference printf()s and exit()s:
 * flash_gemv/csrc/cuda/fuse_gemv_cmp_cuda.cu:25-33,2397-2400). */
int cats_version(void);
const char* cats_status_string(int status);

/* Workspace: scratch for the per-workgroup partial sums, the mask bytes, the fp32 intermediate z and the
 * gate activations of the list-building call.  Replaces the per-call cudaMalloc/cudaFree pairs of the reference
 * (fuse_gemv_cmp_cuda.cu:2351-2354,2402-2403).  The caller allocates cats_workspace_bytes() once (256-byte
 * aligned), runs cats_workspace_init() once (it zero-fills with a kernel), and then passes the same buffer to
 * every call; no call relies on what an earlier call left in it (the counter words at its head are all zero
 * between calls: a call that uses them puts them back).  The size and the carving depend on (H, I)
 * only (B is checked; every region holds what any call of up to CATS_MAX_BATCH rows leaves in it), so one
 * workspace serves every batch size of one layer shape; for another (H, I) use another workspace or initialise
 * again.  One workspace serves one stream at a time. */
size_t cats_workspace_bytes(int B, int H, int I);
int cats_workspace_init(void* ws, size_t ws_bytes, void* stream);

/* Fused gate GEMV + SiLU + |a| > t.  Writes a (B,I) in dtype and/or flag (B,I) bytes; either may be NULL.
 * Replaces fuse_gemv_flag_local / fuse_gemv_flag / fuse_gemv_flag_batch
 * (flash_gemv/flash_gemv/flash_gemv.py:6-7,18-22; fuse_gemv_cmp_cuda.cu:1292-1486,2083-2117). */
int cats_gate_flag(const void* x, const void* wgate, void* a_out, uint8_t* flag_out,
                   int B, int H, int I, int dtype, float threshold, void* stream);

/* Same gate pass, B == 1, that also emits the compact active set: idx_out[0..count) ascending neuron
 * indices (int64), vals_out[0..count) the matching activations in dtype, *count_out (device int32) the
 * count.  Two launches: the gate pass (activations and mask bytes into the workspace), then a small kernel that
 * turns the mask bytes into the list with popcounts, wave prefix sums and bit expansion.
 * Replaces fuse_gemv_cmp (flash_gemv.py:3-4; fuse_gemv_cmp_cuda.cu:43-88,1962-1977), whose list is in
 * atomic arrival order and whose count lives in a process-global managed int. */
int cats_gate_compact(const void* x, const void* wgate, void* vals_out, int64_t* idx_out, int32_t* count_out,
                      int H, int I, int dtype, float threshold, void* ws, size_t ws_bytes, void* stream);

/* Blocking helper for the call above: copies *count_dev to pinned host memory behind the work already on the
 * stream, waits for the stream once and returns the value (or -1 on error). */
int cats_read_count(const int32_t* count_dev, void* stream);

/* Sparse up projection over a flag array.  out[b,j] = flag[b,j] ? a[b,j] * (x[b,:] . wup[j,:]) : 0.
 * Row j of wup is fetched iff any flag[b,j] is set.  a and out are (B,I); out may alias a (in place).
 * out_is_f32 != 0 writes fp32 instead of dtype.
 * Replaces fuse_flag_gemv_local (flash_gemv.py:24-25; fuse_gemv_cmp_cuda.cu:1507-1722,2123-2156) and the
 * Triton gather_gemv_elemul_flag_3d (flash_gemv/flash_gemv/kernels.py:69-254). */
int cats_up_flag(const void* x, const void* wup, const void* a, const uint8_t* flag, void* out, int out_is_f32,
                 int B, int H, int I, int dtype, void* stream);

/* Sparse down projection over neuron-major weights.  y[b,:] += sum_{j: any flag[.,j]} z[b,j] * wdown_t[j,:].
 * z is (B,I) in dtype.  Two output modes:
 *   y_f32 != NULL : fp32 atomics straight into the caller's (B,H) buffer, which the caller zeroed (or wants
 *                   accumulated into) -- atomic_gemv (flash_gemv.py:27-28; fuse_gemv_cmp_cuda.cu:1724-1783,2162-2194);
 *   y_out != NULL : (B,H) in dtype, zero-initialised and rounded inside the call -- the Triton
 *                   gather_transposed_gemv_flag_3d (kernels.py:324-462).
 * Exactly one of y_f32 / y_out must be non-NULL.  Needs a workspace. */
int cats_down_flag(const void* z, const void* wdown_t, const uint8_t* flag, float* y_f32, void* y_out,
                   int B, int H, int I, int dtype, void* ws, size_t ws_bytes, void* stream);

/* Index-list ("DejaVu") up projection: out[b, m] = scale[m] * act(x[b,:] . w[idx[m],:] + bias[idx[m]]) for the M entries
 * of idx (int64 weight-row numbers, any order, duplicates allowed; an entry outside [0, Z) yields 0).  Only the listed
 * rows of w (Z, H) are read.  bias (Z,) and scale (M,) are optional, in dtype; activation 0 = identity, 1 = relu,
 * 2 = squared relu, 3 = swish; fp32 throughout with one rounding at the store.  out (B, M) in dtype.
 * Replaces gather_gemv (flash_gemv/flash_gemv/kernels.py:484-695) and, with scale = the compact gate activations,
 * gather_gemv_elemul_indirect_index_2d (kernels.py:1112-1150, 1236-1274). */
int cats_up_index(const void* x, const void* w, const int64_t* idx, int M, const void* bias, const void* scale, int activation,
                  void* out, int B, int H, int Z, int dtype, void* stream);

/* Index-list down projection: y[b,:] = sum over m of z[b, m] * wdown_t[idx[m], :] (+ bias), z (B, M) aligned with the list,
 * wdown_t (Z, H) neuron-major, bias (H,) optional.  Duplicate entries add up (as the reference's atomics do), entries
 * outside [0, Z) contribute nothing.  y_out (B, H) in dtype, fp32 accumulation in a fixed order.  Needs a workspace.
 * Replaces gather_transposed_gemv (kernels.py:753-1094) and gather_transposed_gemv_indirect_index_2d
 * (kernels.py:1204-1234, 1276-1325). */
int cats_down_index(const void* z, const void* wdown_t, const int64_t* idx, int M, const void* bias, void* y_out,
                    int B, int H, int Z, int dtype, void* ws, size_t ws_bytes, void* stream);

/* Gate + sparse up in one call: out[b,j] = active ? round(a * up) : 0 in dtype, flag_out optional.  One launch; fp32 rows that do not
 * fit on chip from five batch rows on take a dense product each for gate and up, out holding the activations in between.
 * Replaces fuse_gemv_flag_gemv (flash_gemv.py:9-10; fuse_gemv_cmp_cuda.cu:715-784,2006-2022). */
int cats_gate_up(const void* x, const void* wgate, const void* wup, void* out, uint8_t* flag_out,
                 int B, int H, int I, int dtype, float threshold, void* stream);

/* Whole CATS MLP with neuron-major down weights.  1..2 rows: one streaming kernel in which every workgroup takes its
 * neurons through gate, up and down; more rows: gate+up kernel, then sparse down kernel.  Small layers (up to about 13
 * MB a matrix, 23 MB with the partial sums of a batch): one kernel at any number of rows, which reads all rows of all
 * matrices.
 *   y_out != NULL : (B,H) in dtype.  The workgroups leave fp32 partial sums and a second launch adds them in a fixed
 *                   order: the result is bitwise reproducible from run to run.  (The smallest layers at one row, outside
 *                   a stream capture: the last workgroup adds them, in the same order, and there is no second launch.)
 *   y_f32 != NULL : fp32 accumulate into the caller's (B,H), which the caller has zeroed (or which holds what the result
 *                   is to be added to) -- the contract of the reference ops named below.  Everything is added with fp32
 *                   atomics, so calls on different streams, each with a workspace of its own, may add into one buffer.
 *                   At 1..2 rows this is ONE launch, in which every workgroup adds its own sums (the order, and so the
 *                   last bits, vary from run to run); small layers and more rows total their partial sums in a fixed
 *                   order first, in a second launch where the layer needs one, and add each column once.
 * flag_out (B,I) optional.  count_out (device int32, optional) receives the number of neurons active in any row of the
 * batch (the number of neurons fetched; where 9..16 rows run as two passes one small kernel counts the union of the
 * flags afterwards).  With y_f32 and count_out at 1..2 rows a second, tiny launch totals the count.
 * Replaces flag_gemv_gemv_atomic, fuse_gemv_gemv_gemv, fuse_gemv_flag_gemv_gemv (flash_gemv.py:12-16,30-31;
 * fuse_gemv_cmp_cuda.cu:786-1244,2196-2253) and the composite gemv_gemv_triton / flag_gemv_gemv_triton
 * (flash_gemv/flash_gemv/__init__.py:38-48). */
int cats_mlp(const void* x, const void* wgate, const void* wup, const void* wdown_t, void* y_out, float* y_f32,
             uint8_t* flag_out, int32_t* count_out, int B, int H, int I, int dtype, float threshold,
             void* ws, size_t ws_bytes, void* stream);

/* Sparse up + sparse down given the gate activations:  flags = |a| > t per row,  z = a * (x . wup[j]) for active j,
 * y = sum over active j of z[j] * wdown_t[j,:].  Two launches; the flags are derived inside the up kernel and
 * reach the down kernel as mask bytes in the workspace.  a (B,I) in dtype; y_out (B,H) in dtype.
 * Replaces the composite gemv_gemv_triton(x, x_1, Wup, Wdownt, threshold) (flash_gemv/flash_gemv/__init__.py:45-48),
 * the call the reference's sp_method 2 branch makes (experiments/models/sparse_silu/ugly_utils.py:887-894). */
int cats_up_down(const void* x, const void* a, const void* wup, const void* wdown_t, void* y_out, int B, int H, int I,
                 int dtype, float threshold, void* ws, size_t ws_bytes, void* stream);

/* Whole CATS MLP for one row with the gate weight stored (H, I) -- x . wgate_hi, as the reference's index-list and Triton composites
 * take it -- and neuron-major wup, wdown_t (I, H).  Three launches: column sums of the gate pass, then cats_up_down's two, the
 * first of which finishes the activations.  wgate_hi needs the alignment of its element only (any I >= one 16-byte vector).
 * I: at most 2^18 for rows of up to 16 KiB, else 12288 * min(64, 256 / (row bytes / 1024, rounded up)); CATS_ERR_SHAPE beyond what
 * the kernels take, before anything is launched.
 * Replaces flag_gemv_gemv_dejavu and flag_gemv_gemv_triton at one row (flash_gemv/flash_gemv/__init__.py:38-54). */
int cats_mlp_gate_cols(const void* x, const void* wgate_hi, const void* wup, const void* wdown_t, void* y_out, int H, int I,
                       int dtype, float threshold, void* ws, size_t ws_bytes, void* stream);

/* The tail of a decoder layer in two launches:  out = h + MLP(norm_weight * rms_norm(h)).
 * The RMS norm (fp32 mean of squares, rsqrt(mean + eps), result rounded to dtype, then multiplied by norm_weight in
 * dtype -- the HF LlamaRMSNorm / MistralRMSNorm order) is applied while the gate+up kernel stages h in LDS; the
 * residual add happens where the down kernel writes its output (MLP result rounded to dtype first, then added).
 * h, out (B,H) in dtype; out may alias h.  norm_weight (H) in dtype.  Needs B*H*sizeof(dtype) <= 128 KiB.
 * Replaces the three module calls  residual = h; h = post_attention_layernorm(h); h = residual + mlp(h)
 * of the reference's decoder layer (experiments/models/sparse_silu/ugly_utils.py:1036-1057) for batch*seq <= 16. */
int cats_mlp_norm_residual(const void* h, const void* norm_weight, float eps, const void* wgate, const void* wup,
                           const void* wdown_t, void* out, int B, int H, int I, int dtype, float threshold,
                           void* ws, size_t ws_bytes, void* stream);

/* cats_mlp_norm_residual that also writes what the next consumer of the hidden state starts with:
 *   out = h + MLP(norm_weight * rms_norm(h, eps));   next_out = next_norm_weight * rms_norm(out, next_eps).
 * In a decoder stack next_norm_weight is the input_layernorm of the following layer (the final norm after the last
 * layer), so every layer boundary loses its stand-alone norm.  Same two launches: the launch that finishes `out` also
 * leaves each workgroup's finished columns and their sum of squares in the workspace, and per batch row the last of its
 * workgroups to arrive (counters in the workspace head, put back to zero by the call) adds the sums in a fixed order
 * and writes that row of next_out -- bitwise reproducible, +3.4 us on the Llama-2-7B layer.  next_out (B,H) in dtype
 * must not alias out or h.
 * Needs H % 32 == 0 on top of the limits of cats_mlp_norm_residual.
 * Replaces, for batch*seq <= 16, the module calls  residual = h; h = post_attention_layernorm(h); h = residual + mlp(h)
 * of one decoder layer and  hidden_states = self.input_layernorm(hidden_states)  of the next
 * (experiments/models/sparse_silu/ugly_utils.py:1016-1057). */
int cats_mlp_norm_residual_norm(const void* h, const void* norm_weight, float eps, const void* wgate, const void* wup,
                                const void* wdown_t, void* out, const void* next_norm_weight, float next_eps, void* next_out,
                                int B, int H, int I, int dtype, float threshold, void* ws, size_t ws_bytes, void* stream);

/* Whole CATS MLP with the HF (H,I) down weight: gate+up, then a dense row-major GEMV over the zero-filled
 * intermediate (all of wdown is read, as in the reference).
 * Replaces flag_gemv_gemv and flag_gemv_gemv_inner{,_fp32,_bf16} (flash_gemv.py:33-43;
 * fuse_gemv_cmp_cuda.cu:2255-2560). */
int cats_mlp_rowmajor_down(const void* x, const void* wgate, const void* wup, const void* wdown, void* y_out,
                           int B, int H, int I, int dtype, float threshold, void* ws, size_t ws_bytes, void* stream);

/* cats_mlp(y_out mode) for callers that cannot allocate device memory or carry a workspace -- code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc.  It has no counterpart in the reference (whose ops
 * cudaMalloc per call).  The scratch of the single-pass kernels (per-workgroup partial sums and counts, 8 MiB + 4 KiB)
 * lives in a device array inside the library, one copy per GPU, held until the process ends; nothing is allocated or
 * freed by the call.  Limits: 1..2 rows, B * H <= 8192, rows of at most 1024 (one row) or 2048 (two rows) 16-byte
 * vectors (fp32 at one row: H <= 4096); anything else returns CATS_ERR_SCRATCH.  Same kernels (always in two launches) and
 * summation order as cats_mlp, so the same bits.  All calls on one GPU share
 * that GPU's array: calls that overlap in time on one GPU (different streams, or a graph replay next to an eager
 * call) race; calls on one stream, or otherwise ordered, are fine.  Nothing in the array has to be cleared between
 * calls (every call overwrites what it reads). */
int cats_mlp_noalloc(const void* x, const void* wgate, const void* wup, const void* wdown_t, void* y_out,
                     int B, int H, int I, int dtype, float threshold, void* stream);

/* out = x . w^T (+ residual) for 1..8 rows: x (B,K), w (N,K) as nn.Linear holds it, residual and out (B,N), all in dtype.
 * norm_weight (K) != NULL: x is given before its RMS norm, which is applied while x is staged (the norm of
 * cats_mlp_norm_residual).  One rounding, after the residual.  Needs B * K * sizeof(dtype), B rounded up to a power of two and
 * the rows to 8 KiB, to be at most 128 KiB.  The output head and the attention's output projection of a decode step. */
int cats_linear(const void* x, const void* norm_weight, float eps, const void* w, const void* residual, void* out,
                int B, int K, int N, int dtype, void* stream);

/* The attention half of a decoder layer for one new token per row, 1..8 rows, in three launches:
 *   q, k, v = x . W{q,k,v}^T (x normed first if norm_weight is given), rotate-half rotary embedding of q and k at *position, k and v
 *   stored into slot *position of the caches, softmax(q . K^T / sqrt(head_dim)) . V over slots 0..*position, out = h + att . Wo^T.
 * h, x, out (B,H); w* (H,H); caches (B, heads, max_len, head_dim); cos / sin tables (max_len, head_dim); all in dtype.  position: one
 * device word for all rows; outside [0, max_len) nothing is stored and out is NaN.  q_scratch B*H floats, attn_scratch B*H of dtype.
 * head_dim has to be 2..32 (a power of two) 16-byte vectors; the limit on B and H is that of cats_linear.
 * The conventions are those of the reference's decoder layer (experiments/models/sparse_mistral/sparse_silu.py:280-312, 756-832). */
int cats_attention_step(const void* h, const void* x, const void* norm_weight, float eps, const void* wq, const void* wk,
                        const void* wv, const void* wo, void* k_cache, void* v_cache, const void* cos_table, const void* sin_table,
                        const int64_t* position, float* q_scratch, void* attn_scratch, void* out, int B, int H, int heads,
                        int max_len, int dtype, void* stream);

/* ---- a cache of keys and values in 8 bits (fp16 / bf16 models) ----
 * A row has `blocks` blocks of 64 tokens.  A block that is complete is held as e4m3 numbers, with one power of two as scale for a head's keys
 * and one for its values: the smallest s with max |x| <= 448 s over the block's finite values (at least 2^-60; 1 for zeros); each value is x / s,
 * rounded to nearest even, NaN if it is not finite.  The block that holds a row's last token, complete or not, is read as it was given.
 *   k8 (B, kv_heads, blocks, 64, D)   v8 (B, kv_heads, blocks, D, 64)   e4m3, one byte a number
 *   k_scale, v_scale (B, kv_heads, blocks) float       k_tail (B, kv_heads, 64, D)   v_tail (B, kv_heads, D, 64) in dtype, slot = position % 64
 * D is 32, 64, 128 or 256.  k, v and q: strides of a row, a token and a head, in elements, multiples of 8; the elements of a head side by side.
 * start, count: device words, one for each row (step 1) or one for all (step 0).  Row b has min(max(count, 0), T) new tokens (count NULL: T), at
 * positions start .. start + count - 1.  Both calls may be captured; nothing is kept between calls. */
#define CATS_KV8_MAX_BLOCKS (1 << 24)

/* Stores the new tokens: quantises the blocks that they complete and leaves the last block in the tails.  What a row holds already has to end at
 * start (a block's tokens before start are taken from the tails).  So the cache is the same whatever pieces the tokens come in.  Tokens may be taken
 * back by a smaller start, as far as the start of the block that holds the last one, or to the start of any block; what an earlier block held in
 * the type is gone.  To take back drafted tokens that passed a block's end, copy the tails before they are stored, put the copies back, and store the
 * accepted ones again.  Nothing tells a cache from which block its tails are: a start further back makes a wrong block of what they hold.  A row whose tokens do not lie within its blocks is left as it is. */
int cats_kv8_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, const int64_t* start, int start_step,
                    const int64_t* count, int count_step, void* k8, void* v8, float* k_scale, float* v_scale, void* k_tail, void* v_tail, int B,
                    int T, int kv_heads, int D, int blocks, int dtype, void* stream);

/* out[b, i, h] = softmax(scale * q[b, i, h] . K^T) . V over the keys at positions p - window + 1 .. p (window 0: 0 .. p), p = start + i, of cached
 * head h / (heads / kv_heads), for new tokens that cats_kv8_append has stored.  Rows i >= count are zeros; a row whose tokens do not lie within
 * its blocks is NaN.  A query that sees a key or an element of a value that is not finite is NaN (in that element).  out (B, T, heads, D) in
 * dtype, 16-byte aligned.  scale lies in 2^-64 .. 2^64, and scores have to be within 32-bit floats.  Weights are rounded to dtype
 * (their sum is not).  scratch: 16-byte aligned, at least cats_kv8_attention_scratch_bytes() on the device of the call
 * (which may be 0), nothing in it needs to be set.  The reference's attention is that of the models it patches
 * (experiments/models/sparse_mistral/sparse_silu.py:756-832), over a cache in the model's type. */
size_t cats_kv8_attention_scratch_bytes(int B, int T, int heads, int kv_heads, int D, int blocks, int window);
int cats_kv8_attention(const void* q, const int64_t* q_strides, const int64_t* start, int start_step, const int64_t* count, int count_step,
                       const void* k8, const void* v8, const float* k_scale, const float* v_scale, const void* k_tail, const void* v_tail,
                       float scale, int window, void* out, int B, int T, int heads, int kv_heads, int D, int blocks, int dtype, void* scratch,
                       size_t scratch_bytes, void* stream);

/* What cats_kv8_attention launches on the current device, for tests and profiles: plan[0] = 1 where it is the kernel for many tokens, else 0, plan[1] =
 * splits of a row's cache at most.  Not in the reference. */
int cats_kv8_attention_plan(int B, int T, int heads, int kv_heads, int D, int blocks, int window, int* plan);

/* cats_attention_step over such a cache, with as many cached heads as query heads: k and v of the new token go to the tails, and the block that
 * it completes is quantised beside attention.  q is rounded to dtype before the products.  Limits on B and H are those of cats_linear; position lies
 * in [0, max_len), max_len <= 64 * blocks, and what the cache holds ends at it; elsewhere nothing is stored and out is NaN.  Three launches, four
 * where the cache is long enough to be split.  scratch: 256-byte aligned, at least cats_kv8_attention_step_scratch_bytes(), nothing in it needs to be set. */
size_t cats_kv8_attention_step_scratch_bytes(int B, int H, int heads, int blocks);
int cats_kv8_attention_step(const void* h, const void* x, const void* norm_weight, float eps, const void* wq, const void* wk, const void* wv,
                            const void* wo, void* k8, void* v8, float* k_scale, float* v_scale, void* k_tail, void* v_tail, const void* cos_table,
                            const void* sin_table, const int64_t* position, void* out, int B, int H, int heads, int blocks, int max_len, int dtype,
                            void* scratch, size_t scratch_bytes, void* stream);

/* ---- a cache of pages, and packed sequences (fp16 / bf16 models) ----
 * A pool of pages, k_pages and v_pages (pages, kv_heads, page, D) in dtype; page: tokens of a page, a power of two from 16 to 1024.  Token p of sequence s
 * lies in page table[s * table_stride + p / page], place p % page, of the pool.  The table has `width` entries a sequence that are read, and only those of pages
 * that a call needs: the others may be anything.
 * Tokens of a call are packed: sequence s of B has the tokens offsets[s] .. offsets[s + 1] - 1 (none, one or many) of the N tokens of q, k, v and out, at the positions
 * start[s] onwards.  offsets (B + 1) ascend within 0 .. N; tokens before the first and behind the last belong to nobody.  offsets, start, table and shared
 * are read on the device, so a captured call follows them.  D is 32, 64, 128 or 256.  Strides of q, k and v: of a token and of a head, in elements,
 * multiples of 8, a token's at most 2^23; the elements of a head side by side, 16-byte aligned.  All calls may be captured; nothing is kept between calls. */
#define CATS_PAGED_MAX_TOKENS (1 << 24)

/* Stores new tokens, rotated on the way:  x' = x cos[p] + (-x[R/2 .. R-1], x[0 .. R/2-1]) sin[p]  over the first R = rot elements of the heads of q and k, p the
 * token's position, in 32 bits and rounded once; the others, and v, as they are.  cos, sin (positions, rot) in float or in dtype (table_dtype), rot a multiple of 16
 * up to D; rot 0: no rotation, cos and sin are not read.  q, q_out (N, heads, D, contiguous) NULL with heads 0: keys and values only.  A token whose position
 * lies outside the rotary tables or the table's entries, or whose entry is no page, is not stored, and its q_out is NaN; q_out of tokens that are nobody's is zeros.  No two tokens of a call may
 * have one place.  q_out may be q where q is contiguous. */
int cats_paged_append(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                      const int64_t* offsets, const int64_t* start, const void* cos_table, const void* sin_table, int rot, int positions,
                      int table_dtype, void* q_out, void* k_pages, void* v_pages, const int32_t* table, int64_t table_stride, int N, int B, int heads,
                      int kv_heads, int D, int page, int pages, int width, int dtype, void* stream);

/* out[t, h] = softmax(scale * q[t, h] . K^T) . V over the keys at positions p - window + 1 .. p (window 0: 0 .. p), p = start[s] + t - offsets[s], of
 * cached head h / (heads / kv_heads) of the token's sequence s; the new tokens have been stored.  scale lies in 2^-64 .. 2^64, and scores have to be within 32-bit floats.
 * Weights are rounded to dtype (their sum is not): fp16 ones are off by half a step down to 2^-21 of the largest and by 2^-32 of it below that, bf16 ones by half a step
 * down to 2^-86, below which they may be 0.  Products with values are summed in 32 bits, where bf16 weights begin at 2^-40: values below 2^-100 lose bits, and those
 * below 2^-109 may count as 0.
 * group > 1 (B is a multiple of it): each `group` sequences in order have the same first n tokens, n = shared[s / group] (shared_step 1) or shared[0]
 * (shared_step 0), up to start[s] of them for sequence s.  Whole pages of these are read once for all, through the first one's row of the table, whose
 * entries have to be there for them; the page in which they end is each one's own.
 * A sequence whose tokens do not lie within its table's entries is NaN, and so is a query that sees a token whose entry is no page; rows that are nobody's are zeros, and
 * so is a query whose scores are all -infinity.  A query that sees a NaN in a key, or a value that is not finite, is not finite (in that element); a score of -infinity
 * weighs nothing.  Keys that a query does not see, and places behind a sequence's last token, may hold anything.
 * out (N, heads, D), 16-byte aligned.  scratch: 16-byte aligned, at least cats_paged_attention_scratch_bytes() on the device of the call (which may be 0), one for each
 * call that runs at the same time, nothing in it needs to be set.  N * heads / 16 + (B + 2) * kv_heads is below 2^24,
 * and below 2^21 where group > 1. */
size_t cats_paged_attention_scratch_bytes(int N, int B, int heads, int kv_heads, int D, int page, int width, int window, int group);
int cats_paged_attention(const void* q, const int64_t* q_strides, const int64_t* offsets, const int64_t* start, const void* k_pages, const void* v_pages,
                         const int32_t* table, int64_t table_stride, float scale, int window, int group, const int64_t* shared, int shared_step,
                         void* out, int N, int B, int heads, int kv_heads, int D, int page, int pages, int width, int dtype, void* scratch,
                         size_t scratch_bytes, void* stream);

/* The same over keys and values of the call itself, k and v (M, kv_heads, D): sequence s has the keys k_offsets[s] .. k_offsets[s + 1] - 1, and its queries are its
 * last tokens, so that query i of n sees the keys up to i + keys - n.  k_offsets NULL: offsets (M is N), the whole prompt.  A query that sees no key is zeros.
 * M is at least 1. */
int cats_prompt_attention(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                          const int64_t* offsets, const int64_t* k_offsets, float scale, int window, void* out, int N, int M, int B, int heads,
                          int kv_heads, int D, int dtype, void* stream);

/* ---- beam search ---- */
#define CATS_MAX_BEAMS 16

/* The best `keep` continuations of each group of beams:  total(b, v) = scores[b] + logits[b, v] - log sum exp(logits[b, :]), in descending
 * order, equal ones by the lowest b * V + v.  logits (groups, beams, V) in dtype (fp32 too), rows row_stride elements apart; scores (groups, beams)
 * float.  finished (groups, beams) bytes, optional: a beam that has finished goes on only as (b, eos) with its score.  Totals that are not finite
 * count as -infinity (so beams with a score of -infinity take no part).  Outputs (groups, keep): scores, parents (b), tokens (v), and whether a
 * beam has finished (its parent had, or v is eos; eos < 0: none).  Beams are ordered by their logits within a row and by totals in 64 bits between
 * rows, with a sum of 32-bit exponentials (the logarithm is within 2^-21) that goes by the logits alone, wherever a row starts: rows that
 * are the same tie.  keep <= beams * V; both up to CATS_MAX_BEAMS.  scratch: 16-byte aligned, at least cats_beam_scratch_bytes(), nothing in it needs to be set. */
size_t cats_beam_scratch_bytes(int groups, int beams, int V, int keep);
int cats_beam_select(const void* logits, int64_t row_stride, const float* scores, const uint8_t* finished, int64_t eos, float* scores_out,
                     int64_t* parents_out, int64_t* tokens_out, uint8_t* finished_out, int groups, int beams, int V, int keep, int dtype,
                     void* scratch, size_t scratch_bytes, void* stream);

/* Caches moved to the beams that go on, in place: row g * beams + j becomes what row g * beams + parents[g][j] was, in the entries that are live,
 * for each of the n caches.  A cache is (groups * beams, heads, entries) of entry_bytes (a multiple of 4; 16 is faster, on 16-byte boundaries);
 * an entry holds `slots` tokens, and ceil(length / slots) of them are live (slots 0: all are), length being lengths[row of the parent] (step 1) or
 * lengths[0] (step 0).  What is not live stays as it is, and so does a beam whose parent is not within its group.  The caches may not overlap.
 * The array of descriptions is read before the call returns. */
typedef struct {
  void* data;
  int64_t entry_bytes;
  int heads, entries, slots;
} cats_cache_t;
int cats_cache_reorder(const cats_cache_t* caches, int n, const int64_t* parents, const int64_t* lengths, int lengths_step, int groups,
                       int beams, void* stream);

/* z = SiLU(gate) * up over n elements, 0 where |SiLU(gate)| <= threshold; a NaN is kept.  What stands between the matrix products of a
 * prompt in the reference's dense branch (experiments/models/sparse_silu/ugly_utils.py:895-904), with its roundings. */
int cats_silu_mask_mul(const void* gate, const void* up, void* z, size_t n, int dtype, float threshold, void* stream);

/* The whole dense-masked MLP over the M tokens of a prompt (1..CATS_PROMPT_MAX_TOKENS), 16-bit types:
 *   y = (a * (x . Wup^T)) . Wdown^T,  a = SiLU(x . Wgate^T), 0 where |a| <= threshold (a NaN is kept)
 * with the roundings of the three products and of cats_silu_mask_mul.  x (M,H), wgate / wup (I,H), wdown (H,I) at any alignment of the
 * element, H and I at least 8, no matrix of 4 GiB or more; y_out 8-byte aligned.  scratch: 256-byte aligned, at least
 * cats_prompt_scratch_bytes(M, H, I) on the device of the call, nothing in it needs to be set.
 * The reference's dense branch: experiments/models/sparse_silu/ugly_utils.py:895-904. */
#define CATS_PROMPT_MAX_TOKENS 4096
size_t cats_prompt_scratch_bytes(int M, int H, int I);
int cats_prompt_mlp(const void* x, const void* wgate, const void* wup, const void* wdown, void* y_out, int M, int H, int I, int dtype,
                    float threshold, void* scratch, size_t scratch_bytes, void* stream);

/* What cats_prompt_mlp launches for its first product (1, gate and up) or its second (2, down) on the current device, for tests and
 * profiles: plan[0..5] = tile (of kPromptShapes), blocks of tokens, blocks of weight rows, steps a workgroup, ranges of K, steps of loads
 * ahead in registers.  Not in the reference. */
int cats_prompt_plan(int product, int M, int H, int I, int* plan);

/* One launch of cats_mlp(y_out mode) alone, for per-kernel timing and profiling: stage 1 = the streaming launch (gate, up
 * and, for 1..2 rows and small layers, down into per-workgroup partial sums), stage 2 = what finishes y from what stage 1
 * left in the workspace (never one launch with stage 1).  Calling stage 1 then stage 2 with the same arguments is cats_mlp.  Not in the reference. */
int cats_mlp_stage(int stage, const void* x, const void* wgate, const void* wup, const void* wdown_t, void* y_out,
                   int B, int H, int I, int dtype, float threshold, void* ws, size_t ws_bytes, void* stream);

/* Measurement aid, not in the reference: one kernel that reads `bytes` (a multiple of 16, 16-byte aligned) from src
 * with the streaming 128-bit loads the weight rows are read with, and writes nothing (sink, 4 bytes of device memory,
 * is stored to only if the XOR of everything read equals one fixed word).  Timing it over a buffer larger than the
 * 256 MB memory-side cache gives the read-stream bandwidth this GPU actually reaches, the practical ceiling next
 * to the published HBM peak. */
int cats_probe_read(const void* src, size_t bytes, uint32_t* sink, void* stream);

/* Launch-shape knobs for experiments; 0 keeps the built-in choice.  gate_variant N > 0 caps the gate / up kernel at N
 * resident workgroups per CU (N < 0 keeps 3..16 rows off the matrix-core kernels, gate / up and down); down_groups sets the
 * neuron groups of the sparse down kernels, down_block the workgroup size of the wave-per-row-pair one -- and keeps 3..16 rows
 * on that kernel, off the matrix-core one; path 1 keeps the whole-MLP entry points on the separate gate+up
 * and sparse-down kernels for every batch size (by default 1..2 rows take the single-pass kernel).  Any value but 0 (path:
 * 1) keeps whole-MLP calls off the kernels of small layers.  Every setting computes the same function.  Process-global and not synchronised: set it before other threads call in.  Not in the reference. */
int cats_set_tuning(int gate_variant, int down_groups, int down_block, int path);

#ifdef __cplusplus
}
#endif
#endif /* CATS_GEMV_H */
