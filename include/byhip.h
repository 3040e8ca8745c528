/* byhip.h - C ABI of the MI355X (gfx950) backend for BybyLang's quantized tile-GEMM path.
 *
 * libbybyhip.so is the drop-in boundary that a `backends/hip/hip_backend.nim` binds with
 * `importc, cdecl`, the way backends/cpu/cpu_backend.nim:22-26,102-160 binds the CPU C code. Every
 * entry point names the reference interface it replaces (file:line in bobbyshop-vui/bybylang).
 *
 * Conventions (mirroring the reference's native shims):
 *  - Return value: BYHIP_OK (0) on success. BYHIP_UNSUPPORTED (1) is the "false" an encoder
 *    returns for a shape or device it does not handle, after which the caller may take another
 *    route (gpubackend.nim:1444-1445). BYHIP_ERROR (-1) is a failure; byhip_last_error() gives
 *    the message, as nimf_cpu_vm_run_slots fills err/err_len (backends/cpu/cpu_vm.c:178-188).
 *    The library never computes on the CPU: a failure is returned, and the caller's policy
 *    (handleGpuFailure, gpubackend.nim:80-105) decides between raising and its own fallback.
 *  - Memory: device pointers and byte or element counts; no framework types. Work is queued on
 *    the library's stream for the current device and runs asynchronously; results are valid after
 *    byhip_session_end() or byhip_synchronize().
 *  - One host thread drives a session at a time (the reference's global session state,
 *    backends/vulkan/vulkan_driver.nim:1668).
 */
#ifndef BYHIP_H
#define BYHIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define BYHIP_OK 0
#define BYHIP_UNSUPPORTED 1
#define BYHIP_ERROR (-1)

/* Element types of activations and outputs (the reference's session path is fp32 in and out). */
enum byhip_dtype {
    BYHIP_F32 = 0,
    BYHIP_F16 = 1,
    BYHIP_BF16 = 2,
    /* Activations in the FP4-KM packing of the weights: E2M1 nibbles [M, K/2] (byte j of a
     * 32-value group holds element j low and j + 16 high, session_vm.nim:384-388) followed by one
     * E8M0 scale byte per group [M, K/32]. Only byhip_mxfp4_gemm and byhip_fp4km_tile_gemm read
     * it. */
    BYHIP_MXFP4_KM = 3
};

typedef struct byhip_device_info {
    int device;
    int compute_units;
    int wavefront_size;
    int clock_khz;
    int memory_clock_khz;
    int memory_bus_width;
    size_t total_global_mem;
    size_t lds_bytes_per_block;
    char arch_name[64];
    char name[128];
} byhip_device_info;

/* ── Lifecycle and errors ─────────────────────────────────────────────────────────────────── */

/* Selects and initialises `device` (creates the library stream). Replaces the backends'
 * ensureInit / ensureGpuInit (gpubackend.nim detectBackend 131-141; the device ordinal follows
 * BYBY_VULKAN_DEVICE, distributed.nim:144-145, as BYBY_HIP_DEVICE). Idempotent. */
int byhip_init(int device);
int byhip_device_info_get(byhip_device_info* out);
/* Thread-local text of the last failure; "" when none. Backs sessionGetLastError
 * (gpubackend.nim:2647-2667). */
const char* byhip_last_error(void);
void byhip_clear_error(void);
/* The next `count` compute or session entry points fail with "byhip: injected fault" before
 * touching the device, so the host can exercise failure handling (handleGpuFailure,
 * gpubackend.nim:80-105) without a GPU fault. */
void byhip_fault_inject(int count);
int byhip_version(void);

/* ── Device memory ────────────────────────────────────────────────────────────────────────── */

int byhip_alloc(size_t bytes, void** dptr);
int byhip_free(void* dptr);
/* Host -> device copy of `bytes` at byte `dst_off`; stream-ordered. */
int byhip_upload(void* dptr, size_t dst_off, const void* src, size_t bytes);
/* Device -> host copy; waits for the stream first (a read is valid only after the session's
 * work, gpubackend.nim:2669). */
int byhip_read(const void* dptr, size_t src_off, void* dst, size_t bytes);
int byhip_memset(void* dptr, int value, size_t bytes);
int byhip_synchronize(void);
/* The library stream (hipStream_t) of the current device, for callers that time or order their
 * own work against it. */
void* byhip_stream(void);

/* ── Session (gpubackend.nim:894-903 SessionHandle and its lifecycle) ─────────────────────── */

/* sessionBegin (gpubackend.nim:1042): fails if a session is already open
 * (vulkan_driver.nim:1668). */
int byhip_session_begin(void);
/* sessionUpload (gpubackend.nim:1133): a new device buffer holding `n` floats. */
int byhip_session_upload(const float* data, size_t n, void** out);
/* Byte variant (vulkanSessionUploadBytesPrivate, vulkan_driver.nim:2146). */
int byhip_session_upload_bytes(const void* data, size_t bytes, void** out);
/* sessionAllocScratch (gpubackend.nim:1295): `n` floats, zero-filled. */
int byhip_session_alloc_scratch(size_t n, void** out);
/* sessionEnd (gpubackend.nim:2422): waits for the queued work and reports device errors;
 * deferred frees run here (vulkan_driver.nim:1817-1819). */
int byhip_session_end(void);
/* sessionCommitContinue (gpubackend.nim:2444-2467): no wait; the session stays open. */
int byhip_session_commit_continue(void);
/* sessionRecoverQueue (gpubackend.nim:2593): drops an open session after a failed end. */
int byhip_session_recover(void);
/* sessionRead (gpubackend.nim:2669): `n` floats from a session buffer. */
int byhip_session_read(const void* h, float* dst, size_t n);
/* sessionFree (gpubackend.nim:2694): deferred to the end of an open session. */
int byhip_session_free(void* h);
/* sessionGpuSeconds / sessionSetGpuTiming (gpubackend.nim:2617-2632): hipEvent time between
 * begin and end of the timed sessions since the last reset. */
int byhip_session_set_gpu_timing(int on);
double byhip_session_gpu_seconds(void);

/* Record / replay as HIP graphs (gpubackend.nim:2502-2552, vulkan_driver.nim:1659-2030).
 * sessionCanRecord: always 1 on this backend. */
int byhip_session_can_record(void);
/* sessionBeginRecording: opens a session whose queued work is captured; it must be
 * self-contained (entry points that wait for the device, upload or clear memory fail while
 * recording). byhip_session_end() keeps it as a graph, runs it once and waits. */
int byhip_session_begin_recording(void);
/* sessionLastRecording: id kept by the last byhip_session_end(), or -1. */
int byhip_session_last_recording(void);
/* sessionReplay: launches recording `id` `times` times back to back (outside a session), then
 * waits; counted by byhip_session_gpu_seconds() when timing is on. */
int byhip_session_replay(int id, int times);
/* A measurement form of sessionReplay with no counterpart in the reference: launches recording
 * `pre_id` `pre_times` times (untimed), then recording `id` `times` times right behind it, and
 * counts only the latter in byhip_session_gpu_seconds(). All launches are queued before the one
 * wait, so the timed events never include the host's launch latency. */
int byhip_session_replay_after(int pre_id, int pre_times, int id, int times);
/* Measurement marks, with no counterpart in the reference: byhip_session_mark(0) and (1) launch
 * (or, inside a recording, record) a one-thread kernel that stores the GPU's constant-rate
 * realtime counter into the library's begin and end slots. byhip_session_replay_marked(id)
 * launches a recording holding both marks once, waits, and counts the time between the two
 * stores in byhip_session_gpu_seconds() (timing on). Outside recordings and sessions, mark(0)
 * clears the slots before its kernel, and byhip_session_take_marks() waits for the stream and
 * counts the same interval for directly launched work. The slots are the library's: one marked
 * interval at a time. */
int byhip_session_mark(int which);
int byhip_session_replay_marked(int id);
int byhip_session_take_marks(void);
/* sessionFreeRecording. */
int byhip_session_free_recording(int id);
/* A measurement switch with no counterpart in the reference: recordings begun while it is on keep
 * their kernel launches (kernel, launch shape and arguments by value) instead of capturing a HIP
 * graph; ending one launches them in order, and every replay launches them again, directly on the
 * library stream. Same results as the graph form; it exists so that profilers which trace direct
 * dispatches see exactly the replayed kernels (off by default). */
int byhip_session_set_direct_replay(int on);

/* ── Q4 block-dequant GEMV / GEMM ─────────────────────────────────────────────────────────── */

/* Resident Q4 weights: the ResidentWeightHandle of gpubackend.nim:2813-2825. */
typedef struct byhip_q4w byhip_q4w;

typedef struct byhip_q4w_info {
    int K, N, group_size, groups_per_row;
    int scale_is_f16;   /* scales held as fp16 (every scale was exactly representable) */
    int zero_uniform;   /* one zero point for every group (its value in zero_value) */
    float zero_value;
    size_t device_bytes;
    /* every (q - zero) * scale lies in fp16's normal range (or is 0): the fp16 MFMA kernels may
     * take these weights at M > 8; otherwise the exact fp32 GEMM does */
    int f16_safe;
} byhip_q4w_info;

/* residentUploadQ4 (gpubackend.nim:2883-2919) and residentUploadQ4Mapped (2961-2998): host wq
 * (`wq_bytes` bytes, the packed rows [N, (K+1)/2] start at byte `wq_off`; even k in the low
 * nibble), scales and zeros fp32 [N * groups_per_row]. The weights are copied once into the device
 * layout (fp16 scales when exact, one zero when uniform). group_size 0 means one group per row,
 * as in cpu_kernels_impl.inc:309. */
int byhip_q4_resident_upload(const uint8_t* wq, size_t wq_bytes, size_t wq_off,
                             const float* scales, const float* zeros, int K, int N,
                             int group_size, int groups_per_row, byhip_q4w** out);
/* The same from device-resident fp32 scale/zero arrays and nibble rows (e.g. session buffers). */
int byhip_q4_resident_from_device(const void* d_wq, size_t wq_off, const void* d_scales,
                                  const void* d_zeros, int K, int N, int group_size,
                                  int groups_per_row, byhip_q4w** out);
/* residentFreeQ4 (gpubackend.nim:3233-3253). */
int byhip_q4_resident_free(byhip_q4w* w);
int byhip_q4_resident_info(const byhip_q4w* w, byhip_q4w_info* out);

/* sessionMatmulQ4 (gpubackend.nim:3000-3061): y[M, N] = x[M, K] . W^T on device buffers,
 * computing sum_k x[m,k] * (q[n,k] - zero[n,g]) * scale[n,g] (cpu_kernels_impl.inc:293-319,
 * cpu_vm.c:420-482) with fp32 accumulation. x_dtype: BYHIP_F32 or BYHIP_F16; y_dtype: BYHIP_F32,
 * BYHIP_F16 or BYHIP_BF16. M <= 8 runs the decode GEMV; larger M the fp16 MFMA GEMMs when the
 * weights are fp16-safe (byhip_q4w_info.f16_safe), else the exact fp32 GEMM. fp32 activations
 * keep the reference's fp32 tolerance on every route (1e-4 of max(1, |y|max)); fp16 activations
 * at M > 8 use weights rounded once to fp16. */
int byhip_q4_matmul(const void* x, int x_dtype, const byhip_q4w* w, void* y, int y_dtype, int M);

/* No counterpart in the reference: byhip_q4_matmul for callers that cannot allocate device memory
 * (code under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc). Same
 * arguments, kernels and results; tuned plans are not consulted. The kernels' scratch (split-K
 * partial sums, per-row shifts of fp32 activations) is a 16 MiB device array inside the library,
 * one per GPU, set up by byhip_init: the call allocates nothing. More than 4,194,304 rows of fp32
 * activations at M > 8 are rejected (BYHIP_ERROR). Calls on one GPU share the array: calls that
 * overlap (other threads or streams) race on it. */
int byhip_q4_matmul_static(const void* x, int x_dtype, const byhip_q4w* w, void* y, int y_dtype, int M);

/* residentPrepareQ4 (gpubackend.nim:2871-2880; vulkanPrepareQ4Tuned, q4_autotune.nim:387-543):
 * chooses the kernel byhip_q4_matmul uses for these weights, this M's class (1; 2..32; 33..128;
 * more, tuned at M = 1, 32, 64 and 256) and activation dtype (BYHIP_F32 is the reference's session
 * dtype).
 * Every candidate runs once on deterministic input and must match the exact per-element kernel
 * within 1e-4 of the output's magnitude (3e-3 for kernels that round weights to fp16 for the MFMA)
 * with finite outputs; the survivors are timed and the fastest by at least 3% is kept, in memory
 * and in a plan file under BYHIP_CACHE_DIR (else $XDG_CACHE_HOME/bybylang_amd or
 * ~/.cache/bybylang_amd) keyed by the device and the library's kernel sources, so a later process
 * reuses it (q4_autotune.nim:32-50). Returns BYHIP_UNSUPPORTED when tuning is off
 * (BYHIP_Q4_TUNED=0 or BYHIP_GPU_AUTOTUNE=0) or a session is open, as the reference does. */
int byhip_q4_prepare(const byhip_q4w* w, int M, int x_dtype);
/* The plan in place for these weights, M class and dtype: its name and whether it came from the
 * plan file (1) or was tuned in this process (0); BYHIP_UNSUPPORTED when there is none. */
int byhip_q4_plan_info(const byhip_q4w* w, int M, int x_dtype, char* name, int name_len, int* from_cache);
/* Forgets this process's plans (the plan file stays; the next prepare reads it again). */
int byhip_q4_plans_reset(void);

/* sessionMatmulQ4Fused (gpubackend.nim:3185-3231; its shader, q4_autotune.nim:194-330): the fused
 * decode GEMV, M = 1, on fp32 device buffers.
 *   mode 0: ws[0..n_ws-1] (1..3 resident weights of equal K, group and groups per row) share `a`
 *           (K floats); outs[i] receives ws[i]'s N rows.
 *   mode 1: ws = {gate, up} of equal N; outs[0][row] = silu(gate . x) * (up . x), with
 *           silu(v) = v / (1 + exp(-v)). As in the reference, outs holds an allocated buffer per
 *           weight (n_outs >= 2); only outs[0] is written.
 *   has_norm: `a` is the raw vector; RMSNorm with weights `gamma` (K floats) and `eps` is applied
 *           inside the kernel: x = a * gamma, each dot product times 1 / sqrt(sum a^2 / K + eps).
 *   has_res: res[row] (matrix-local row) is added to each output.
 * Returns BYHIP_UNSUPPORTED, with the outputs untouched, for the combinations the reference's
 * encoders reject (n_ws outside 1..3, n_outs < n_ws, mode 1 without exactly two weights, a missing
 * output, residual or norm buffer) and for weights this kernel does not take (mismatched shapes
 * or scale formats, K % 32 != 0); any K that is a multiple of 32 is taken (long rows in K slices).
 * The caller then runs the unfused sequence, as the reference's callers do. */
int byhip_q4_matmul_fused(int mode, const float* a, byhip_q4w* const* ws, int n_ws, float* const* outs,
                          int n_outs, const float* res, int has_res, const float* gamma, float eps,
                          int has_norm);
/* gpuMatmulQ4 (gpubackend.nim:806-843): host fp32 in, host fp32 out; uploads the weights on every
 * call and waits, like vulkanMatmulQ4 (vulkan_driver.nim:1012-1161). */
int byhip_gpu_matmul_q4(const float* a, const uint8_t* wq, const float* scales, const float* zeros,
                        float* c, int M, int K, int N, int group_size, int groups_per_row);

/* ── FP4-KM tile GEMM and MXFP4 ───────────────────────────────────────────────────────────── */

/* OP_TILE_GEMM format 0 (cpu_vm.c:583-628, tile_gemm.nim:1-26): y[M, N] = x[M, K] . W^T with W
 * the FP4-KM blob in `blob` (nibbles [N, K/2] from byte 0, scale bytes [N, K/32] from byte
 * `scale_base`) and the 272-float decode table at float `lut_base` of `lut` (16 FP4 values, then
 * 256 scale values): weight = lut[nibble] * lut[16 + scale byte]. x_dtype BYHIP_F32 / BYHIP_F16,
 * or BYHIP_MXFP4_KM when the table is exactly E2M1 and 2^(e-127) (then the native scaled MFMA runs;
 * otherwise BYHIP_UNSUPPORTED). `blob_bytes` and `lut_floats` bound the reads as the CPU VM bounds
 * them (cpu_vm.c:600-604). Replaces sessionFp4GemmTensorCore / sessionFp4GemmTiledEnc /
 * sessionFp4GemmMetal (gpubackend.nim:1442-1472). */
int byhip_fp4km_tile_gemm(const void* x, int x_dtype, const uint8_t* blob, size_t blob_bytes,
                          size_t scale_base, const float* lut, size_t lut_floats, size_t lut_base,
                          void* y, int y_dtype, int M, int K, int N);
/* Native MXFP4 GEMM (the FP4 configuration of the benchmark): x and w both in the FP4-KM packing
 * with E8M0 scale bytes (x: nibbles [M, K/2] then scales [M, K/32]; w: nibbles [N, K/2] then scales
 * [N, K/32] at byte N*K/2), E2M1 values, fp32 accumulation, y_dtype F32/F16/BF16. */
int byhip_mxfp4_gemm(const uint8_t* x, const uint8_t* w, void* y, int y_dtype, int M, int K, int N);
/* OP_TILE_GEMM format 1 (cpu_vm.c:550-582): W IEEE halves [N, K]; sessionF16GemmTile
 * (gpubackend.nim:1474-1481). */
int byhip_f16_tile_gemm(const void* x, int x_dtype, const uint16_t* w, size_t w_halves,
                        void* y, int y_dtype, int M, int K, int N);
/* sessionTileGemmReady (gpubackend.nim:1483-1488, vulkanTileGemmReady vulkan_driver.nim:2681-2762):
 * the parity gate on closed-form data whose sums are exact, run once per process and format;
 * returns 1 (passed), 0 (failed) or BYHIP_ERROR. `tensor_core` selects the MFMA route. */
int byhip_tile_gemm_ready(int f16, int tensor_core);

/* ── Micro-VM route (session_vm_dispatch.nim:128-158, slot_layout.nim:11-73) ───────────────── */

/* Runs a shape-op micro-kernel program on the five slots the reference binds (mem, u8, lut,
 * input, u32; slot_layout.nim:23-37): OP_TILE_GEMM (formats 0 and 1), OP_FP4_COOP_GEMM,
 * OP_Q4_GEMV and OP_Q4_COOP_GEMM, decoded with the rules of nimf_cpu_vm_run_slots
 * (cpu_vm.c:420-628) and tileGemmShape (tile_gemm.nim:68-78). Slots are device pointers; lengths
 * are in the reference's units (mem, lut, input: floats; u8: bytes). `rows` > 0 overrides an
 * M = 0 header (a dispatch's row count); with rows = 0, M = 0 means input_len / K. A rejected
 * program returns BYHIP_ERROR with the reference's own message ("CPU VM unsupported tile GEMM
 * (format 0 K 48 N 16)", "CPU VM q4_coop_store out of range: 64", ...), checked in its order, and
 * leaves in `mem` the outputs the reference writes before it stops. The Q4 shape ops run the exact
 * routes (fp32 arithmetic, as in the reference). The program's remaining words may only be tile
 * ops, barriers, NOPs and HALT (else BYHIP_UNSUPPORTED). */
int byhip_program_dispatch(const uint32_t* words, int n_words, void* mem, size_t mem_len,
                           const void* u8, size_t u8_len, const void* lut, size_t lut_len,
                           const void* input, size_t input_len, int rows);

/* ── Attention over a paged cache ─────────────────────────────────────────────────────────────
 *
 * The half of a decoder layer between the QKV and the O projection, and the norms around it, with no
 * counterpart in the reference's backends. Everything lives on the device: the cache, the page tables,
 * the lengths and the reference counts, so a step that grows, forks or frees sequences can be recorded
 * with the calls that use them. Kernels check every page id, row and position they take from device memory
 * against the sizes given here and leave out what lies outside. */

/* One layer's cache, in the caller's memory: keys and values each [pages][kv_heads][page_size][head_dim],
 * dtype BYHIP_F16 or BYHIP_BF16. */
typedef struct byhip_kv_cache {
    void* k;
    void* v;
    int dtype;
    int pages, page_size, kv_heads, head_dim;
} byhip_kv_cache;

/* The sequences of a call. Sequence b holds lens[b] tokens, this call's own among them, in pages
 * table[b * table_stride ..]; this call's rows starts[b] .. starts[b + 1] - 1 are its last tokens, so row i of
 * them has position lens[b] - (starts[b + 1] - starts[b]) + i. Device arrays; starts[0] = 0, ascending,
 * at most `rows`: a sequence whose rows pass them is left out. */
typedef struct byhip_kv_batch {
    const int* table;
    const int* starts;  /* [batch + 1] */
    const int* lens;    /* [batch] */
    int batch, table_stride, rows;
    const int* granted; /* [batch] or NULL: tokens that sequence b's last cache_grow got (byhip_kv_pool). Where it brings more
                         * rows than that, they have no position: nothing is appended for them, and their attention is 0. A
                         * caller whose grows may be refused passes it: lens then does not count the refused rows, and without
                         * it they would take the places of the tokens before them, in pages that others may share. */
} byhip_kv_batch;

enum byhip_rope_layout {
    BYHIP_ROPE_HALVES = 0,  /* value i turns with value i + rot_dim / 2 */
    BYHIP_ROPE_PAIRS = 1    /* value 2 i turns with value 2 i + 1 */
};
enum byhip_rope_scaling {
    BYHIP_ROPE_PLAIN = 0,   /* turns per position base^(-2 i / rot_dim) / (2 pi) */
    BYHIP_ROPE_LINEAR = 1,  /* the same over `factor` (position interpolation) */
    BYHIP_ROPE_BASE = 2,    /* base * factor^(rot_dim / (rot_dim - 2)): the slowest pair slows by `factor` */
    BYHIP_ROPE_PARTS = 3    /* pairs that turn fewer than `slow` times in original_len positions slow by
                             * `factor`, those of more than `fast` turns stay, a ramp linear in the turns between;
                             * magnitude 0.1 ln(factor) + 1. (A model that was trained with a ramp linear in the
                             * pair's index needs steps of the caller's own.) */
};
/* Rotary positions of the first rot_dim values of a head (even; the others pass through): steps[i] (device,
 * rot_dim / 2) is pair i's turn per position in units of 2^-64 of a whole turn, so that position * step
 * modulo 2^64 is the angle at any position without rounding. Rotated values are multiplied by `magnitude`. */
typedef struct byhip_rope {
    int layout;
    int rot_dim;
    float magnitude;
    const uint64_t* steps;
} byhip_rope;

/* Fills steps[rot_dim / 2] and *magnitude (host memory) for a base and scaling. Needs no device. */
int byhip_rope_steps(int rot_dim, double base, int scaling, double factor, double original_len, double slow,
                     double fast, uint64_t* steps, float* magnitude);

/* Rotary positions and the cache's append in one pass: rows of `heads` query heads, kv_heads key heads and
 * kv_heads value heads (x_dtype F32 / F16 / BF16, row strides in elements, so the three may lie in one QKV
 * buffer). The rotated queries go to q_out; rotated keys and values go to their positions in the
 * cache's pages, rounded once to its dtype. rope NULL: no rotation. cache NULL: queries only (k, v unused;
 * head_dim then comes from `head_dim`, which otherwise must be 0 or the cache's). q_out may be q itself where
 * the types and strides agree. */
int byhip_rope_append(const void* q, size_t q_stride, const void* k, size_t k_stride, const void* v,
                      size_t v_stride, int x_dtype, int heads, int head_dim, const byhip_rope* rope,
                      const byhip_kv_cache* cache, const byhip_kv_batch* batch, void* q_out,
                      size_t q_out_stride, int q_out_dtype);

/* How scores become weights: s = scale * q . k; softcap > 0: s = softcap * tanh(s / softcap); slopes
 * (device, [heads], or NULL): s -= slopes[head] * |position - j|. Key j < lens[b] is seen from position p where
 * j <= p and (window <= 0 or p - j < window), or j < prefix[b] (device, [batch], or NULL). */
typedef struct byhip_attn {
    float scale;
    float softcap;
    int window;
    const float* slopes;
    const int* prefix;
} byhip_attn;

/* Attention of the call's rows (a token each, a chunk, or any mixture) over the cache: q and out are rows of
 * `heads` heads (heads % kv_heads == 0, neighbouring heads share a key head). Rows that see no key, or
 * whose scores are all -inf, give zeros; what the masks hide has no influence, whatever it holds.
 * q_dtype F32, or the cache's dtype; out_dtype F32, F16 or BF16. fp32 on either side keeps fp32's
 * precision throughout; with 16-bit q and out the weights are rounded once to the cache's dtype before they
 * multiply the values. Sums and softmax statistics are fp32. */
int byhip_paged_attention(const void* q, size_t q_stride, int q_dtype, int heads, const byhip_attn* attn,
                          const byhip_kv_cache* cache, const byhip_kv_batch* batch, void* out,
                          size_t out_stride, int out_dtype);

/* The pages of all layers' caches (a host array of descriptors of equal geometry), which share one page table:
 * sequence slot r holds lens[r] tokens in pages table[r * table_stride ..]; refs[p] counts the slots that
 * hold page p (0: free). All device arrays. status (device, 4 ints, cleared by the caller) adds up over
 * calls: [0] slots refused for want of pages or table columns, [1] entries refused as invalid (a slot or parent out of
 * range or named twice), [2] pages copied, [3] pages newly taken. A refused entry changes nothing else but granted
 * (device, [slots], or NULL): cache_grow writes there how many tokens a slot got, 0 where it was refused or shrank. */
typedef struct byhip_kv_pool {
    const byhip_kv_cache* caches;
    int n_caches;
    int* refs;
    int* table;
    int* lens;
    int slots, table_stride;
    int* status;
    int* granted;
} byhip_kv_pool;

/* Slot rows[i] becomes a fork of slot parents[i]: what it held is released, the parent's pages are shared. A
 * parent that is itself among `rows` is refused. n <= 1024. */
int byhip_cache_fork(const byhip_kv_pool* pool, const int* parents, const int* rows, int n);
/* Slots rows[i] release their pages; their lengths become 0. n <= 1024. */
int byhip_cache_free(const byhip_kv_pool* pool, const int* rows, int n);
/* Slot rows[i] gets room for add[i] more tokens and counts them in lens: the lowest free pages, in the
 * order of i. A negative add[i] drops that many tokens (at most all) and releases the pages that then hold none. A partly filled last page that others still hold is copied first, so that a slot only ever
 * appends to pages of its own. Slots past the first that does not fit are refused. n <= 1024. */
int byhip_cache_grow(const byhip_kv_pool* pool, const int* rows, const int* add, int n);
/* Moves live pages to the front: the i-th free page below the number of live ones receives the i-th live page
 * above it. refs and all tables follow; refs_out / table_out (or NULL: in place) receive them. */
int byhip_cache_compact(const byhip_kv_pool* pool, int* table_out, int* refs_out);
/* Page src[i] of every layer is copied to page dst[i] (device arrays; no dst twice or among src; pairs
 * outside the pool are left out). */
int byhip_cache_copy(const byhip_kv_pool* pool, const int* src, const int* dst, int n);

enum byhip_norm_kind { BYHIP_NORM_RMS = 0, BYHIP_NORM_LAYER = 1 };
/* v / sqrt(mean(v^2) + eps), or (v - mean) / sqrt(variance + eps); then * weight + bias (device, fp32, each
 * may be NULL). */
typedef struct byhip_norm {
    int kind;
    float eps;
    const float* weight;
    const float* bias;
} byhip_norm;

/* Between two blocks, M rows of N values: h = res_scale * res + gate * post(x), y = pre(h). post NULL: x
 * itself; gate (fp32, gate_stride between rows, 0: one row for all) NULL: 1; res NULL: 0; h NULL: not
 * stored; pre NULL: no y. res and h have h_dtype and may be the same rows. y is formed from h before its rounding.
 * Row strides in elements. */
int byhip_norm_block(const void* x, size_t x_stride, int x_dtype, int M, int N, const byhip_norm* post,
                     const float* gate, size_t gate_stride, const void* res, size_t res_stride,
                     float res_scale, void* h, size_t h_stride, int h_dtype, const byhip_norm* pre, void* y,
                     size_t y_stride, int y_dtype);

/* ── Debug (bit-exact unpack checks) ──────────────────────────────────────────────────────── */

/* Unpacks resident Q4 weights on the device into host arrays: codes [N*K] (0..15), scales and
 * zeros [N * groups_per_row] as fp32, from the device layout. */
int byhip_debug_unpack_q4(const byhip_q4w* w, uint8_t* codes, float* scales, float* zeros);
/* Unpacks an FP4-KM blob on the device: codes [N*K] in element order (k), decoded weights
 * [N*K] = lut[code] * lut[16 + scale byte] as fp32. */
int byhip_debug_unpack_fp4km(const uint8_t* blob, size_t scale_base, const float* lut,
                             size_t lut_base, int K, int N, uint8_t* codes, float* weights);
/* A plain device copy of `bytes` (16-byte multiples): the reference point for HBM bandwidth and
 * for scaling hardware traffic counters. No counterpart in the reference. */
int byhip_debug_copy(void* dst, const void* src, size_t bytes);
/* A plain streaming read of `bytes` (16-byte multiples; nontemporal 16-byte loads, eight per lane
 * in flight, 16 waves per CU): the reference point for what the kernels' reads can reach. Each
 * wave stores a fold of what it read into `sink`, which must hold 16 * CUs 32-bit words.
 * No counterpart in the reference. */
int byhip_debug_read(const void* src, size_t bytes, void* sink, size_t sink_bytes);
/* The number of device allocations the library has made since the process started (its buffers,
 * resident weights, workspace and internal temporaries): a test checks with it that an entry
 * point allocates nothing. No counterpart in the reference. */
unsigned long long byhip_debug_alloc_count(void);

#ifdef __cplusplus
}
#endif
#endif
