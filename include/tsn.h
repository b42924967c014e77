/* tsn.h — C ABI of the B200 (sm_100a) MMDiT denoising path of thinksound-native.
 *
 * Three faces, each replacing one layer of the reference (paths relative to the reference repo):
 *   device face   tsn_device_* / tsn_alloc / tsn_dispatch / tsn_commit   -> src/gpu.h Device (src/gpu.mm)
 *   runtime face  tsn_gemm / tsn_gemv / tsn_conv / tsn_cfg_euler ...     -> src/net.h Runtime (src/net.mm)
 *   model face    tsn_dit_*                                              -> src/models.h DitModel
 *                 (src/dit.cpp, src/dit_fwd.cpp) and the sampler loop of src/pipeline.cpp:126-155
 *
 * Conventions: every call returns TSN_OK (0) or a TSN_ERR_* code; tsn_last_error() gives the
 * message of the last failure on the calling thread. Pointers named *_dev are device (or
 * managed) addresses; *_host are host addresses; "any" pointers may be either (cudaMemcpyDefault).
 * All work is issued on the device's stream (tsn_device_set_stream); calls that return results to
 * the host synchronise that stream. No entry point falls back to the CPU: without a usable
 * sm_100 device every compute call fails with TSN_ERR_CUDA.
 */
#ifndef TSN_H
#define TSN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
    TSN_OK = 0,
    TSN_ERR_ARG = 1,          /* bad argument or unsupported geometry */
    TSN_ERR_CUDA = 2,         /* CUDA runtime/driver error, or no usable device */
    TSN_ERR_IO = 3,           /* file not found / unreadable */
    TSN_ERR_FORMAT = 4,       /* malformed GGUF */
    TSN_ERR_MISSING = 5,      /* a tensor the DiT needs is absent or mis-shaped */
    TSN_ERR_OOM = 6,          /* device allocation failed */
    TSN_ERR_UNSUPPORTED = 7,  /* kernel name or mode not provided by this build */
    TSN_ERR_TIMEOUT = 8,      /* a device-side wait gave up (kernel reported through the error word) */
    TSN_ERR_STATE = 9         /* call out of order (e.g. forward before prepare) */
};

/* Operand type of the tensor-core GEMMs. F16 matches the reference's device weights
 * (BF16 GGUF values converted with the reference's f32->f16 rule, src/net.mm:141-168). */
enum { TSN_COMPUTE_F16 = 0, TSN_COMPUTE_BF16 = 1 };

const char * tsn_last_error(void);
int tsn_version(void);

/* ------------------------------------------------------------------ device face (src/gpu.h) */
typedef struct tsn_device tsn_device;

/* Device::init (src/gpu.h:25). Binds CUDA device `ordinal`; creates a private stream. */
int tsn_device_create(int ordinal, tsn_device ** out);
/* Device::~Device (src/gpu.h:22). Frees every buffer tsn_alloc returned (the reference has no free). */
int tsn_device_destroy(tsn_device * dev);
/* Use an external cudaStream_t (e.g. the caller's framework stream) for all later work. */
int tsn_device_set_stream(tsn_device * dev, void * cuda_stream);
void * tsn_device_stream(tsn_device * dev);
/* Device::alloc (src/gpu.h:26, src/gpu.mm:52-64): zeroed managed memory, so the pointer is
 * valid on host and device like the reference's unified-memory Buf.p. 0 bytes -> 16 bytes. */
int tsn_alloc(tsn_device * dev, size_t bytes, void ** out);
/* Device::wrap (src/gpu.h:28, src/gpu.mm:66-87): register caller memory without copying. */
int tsn_wrap(tsn_device * dev, const void * p, size_t bytes, void ** out);
/* Device::begin (src/gpu.h:31). */
int tsn_begin(tsn_device * dev);
/* Device::dispatch (src/gpu.h:34-38): run the reference kernel `kernel` by name with its Metal
 * param block. grid/block are advisory (Metal threadgroup semantics); each kernel uses its own
 * CUDA launch geometry. Unknown names -> TSN_ERR_UNSUPPORTED (the reference logs and skips). */
int tsn_dispatch(tsn_device * dev, const char * kernel, const uint32_t grid[3], const uint32_t block[3],
                 const void * const * bufs, int nbufs, const void * params, size_t nparams);
/* Device::commit (src/gpu.h:39): synchronise the stream; records the queue time for last_gpu_ms. */
int tsn_commit(tsn_device * dev);
/* Device::exec_width (src/gpu.h:40): 32 for every provided kernel, 0 for unknown names. */
uint32_t tsn_exec_width(tsn_device * dev, const char * kernel);
/* Device::last_gpu_ms (src/gpu.h:41). */
double tsn_last_gpu_ms(tsn_device * dev);
/* No counterpart in the reference (a test hook for the failure path). Launches one block whose
 * thread waits on an mbarrier that nothing ever arrives on, bounded by limit_us (100 us .. 1 s), the
 * way every pipeline wait of this library is bounded. Expected result: TSN_ERR_TIMEOUT, with the
 * device still usable afterwards. */
int tsn_selftest_device_timeout(tsn_device * dev, uint32_t limit_us);
/* No counterpart in the reference (a test hook for an experimental GEMM, not used by any model
 * path). Y[M,N] = X·W^T (+bias) with X f32 [M][K], W f16 [N][K], Y f32 [M][N]. mode 0: X split into
 * an f16 high part on the f16 tensor path and its residual, scaled by 2^12, as e4m3 against an e4m3
 * copy of W scaled by 2^wexp (tile width bn 128, 176 or 256); mode 1: the library's split f16 GEMM
 * (bn 128 or 256); modes 2 and 3: a split f16 GEMM with K blocks of 64 or 32, so twice the stages
 * (bn 128, 176 or 256); mode + 4: the same without the L2-evicting write between launches. Operands are
 * prepared outside the timing; each of reps launches (1..100) is timed alone, and *ms (may be null)
 * receives the mean. K a multiple of 64.
 * Allocates its scratch; synchronises. */
int tsn_selftest_gemm_lo8(tsn_device * dev, const void * W, const void * X, void * Y, const void * bias, uint32_t M,
                          uint32_t N, uint32_t K, int wexp, int mode, int bn, int reps, float * ms);
/* No counterpart in the reference (a test hook for the batched GEMV that carries the t-embedding
 * and every clip/text modulation of a step; each job is one Runtime::gemv, src/net.mm:51-56).
 * njobs jobs (1..64), job q: Y_q[b][n] = act(sum_k W_q[n][k] x[b][k] + bias_q[n]) for b < nb,
 * n < N[q]; act 0 none, 1 SiLU. W: the jobs' f16 rows of K back to back (job q from row sum N[<q]);
 * bias: f32, laid out the same way, or null; x: [nb][K] f32; Y: [nb][sum N] f32, job q's arm b at
 * b * sum N + sum N[<q]. K a multiple of 8 up to 1024; nb <= nb_cap <= 8 (the kernel instance's arm
 * capacity); blocks: the grid's cap (>= 1; results do not depend on it). tc = 1: the tensor-core form
 * the model uses for its modulation jobs (K a multiple of 64, act 0, at most 16 jobs; nb_cap unused).
 * Synchronises. */
int tsn_selftest_gemv_jobs(tsn_device * dev, const void * W, const void * bias, const void * x, void * Y,
                           const uint32_t * N, int njobs, uint32_t K, int nb, int nb_cap, int act, int blocks, int tc);

/* ------------------------------------------------------------------ runtime face (src/net.h) */
/* Runtime::gemm (src/net.h:23-24): Y[M,N] = X[M,K]·W[N,K]^T (+bias), X/Y f32, W f16 (wf16=1) or
 * f32 (wf16=0), leading dimensions in elements (0 = dense). */
int tsn_gemm(tsn_device * dev, int wf16, const void * W, const void * X, void * Y, const void * bias,
             uint32_t M, uint32_t N, uint32_t K, uint32_t ldx, uint32_t ldw, uint32_t ldy);
/* No counterpart in the reference. The same product as tsn_gemm with f16 weights, for callers
 * that must not allocate device memory once running: an audio host's real-time render thread
 * (cudaMalloc can take a device-wide lock and synchronise the GPU mid-callback) or a process
 * whose device memory another framework's pool allocator divided up front. tsn_gemm grows a
 * cudaMalloc'd scratch buffer for its split f16 copy of X; this entry point uses a fixed 8 MiB
 * device array inside the library instead and calls no allocator. Limits: K and N multiples of
 * 64, and 4*M*K bytes (plus 2*N*K when ldw != K) at most 8 MiB, else TSN_ERR_ARG. The first call
 * on each device looks up the array's device address; make that first call before any stream
 * capture begins; the looked-up address does not survive cudaDeviceReset of that device. Every
 * call on a device shares the one array: calls that overlap on the GPU (other streams, other
 * threads) race on it, so serialise them. */
int tsn_gemm_noalloc(tsn_device * dev, const void * W, const void * X, void * Y, const void * bias,
                     uint32_t M, uint32_t N, uint32_t K, uint32_t ldx, uint32_t ldw, uint32_t ldy);
/* Runtime::gemv (src/net.h:25-26). */
int tsn_gemv(tsn_device * dev, const void * W, const void * X, void * Y, const void * bias,
             uint32_t N, uint32_t K, uint32_t ldw, int wf16);
/* Runtime::conv (src/net.h:29-31): conv1d of x [T,IC] with W (GGUF [K,IC,OC], i.e. [OC][IC][K]). */
int tsn_conv(tsn_device * dev, int wf16, const void * W, const void * bias, const void * x, void * y,
             uint32_t T, uint32_t OL, uint32_t IC, uint32_t OC, uint32_t K, uint32_t stride, uint32_t pad,
             uint32_t dil, int convt);
/* Runtime elementwise helpers (src/net.h:36-48). */
int tsn_silu(tsn_device * dev, void * x, size_t n);
int tsn_copy(tsn_device * dev, const void * x, void * y, size_t n);
int tsn_swiglu(tsn_device * dev, const void * a, const void * b, void * y, size_t n);
int tsn_add(tsn_device * dev, const void * a, const void * b, void * y, size_t n);
int tsn_add_bcast_col(tsn_device * dev, const void * x, const void * v, void * y, uint32_t S, uint32_t H);
/* Runtime::cfg_euler (src/net.h:46-47): x += dt·(fu + cfg·(fc − fu)). */
int tsn_cfg_euler(tsn_device * dev, const void * fc, const void * fu, void * x, size_t n, float cfg, float dt);
int tsn_mean_cols(tsn_device * dev, const void * x, void * y, uint32_t S, uint32_t H);

/* ------------------------------------------------------------------ model face (src/models.h) */
typedef struct tsn_dit tsn_dit;

typedef struct tsn_dit_geom {
    uint32_t H, NH, F, depth, fused_depth, latent_dim;
    float rope_theta, t_max_period;
} tsn_dit_geom;

/* DitModel::load (src/models.h:67, src/dit.cpp:29-46): read the GGUF, upload its BF16 tensors to
 * HBM and convert them there (qkv rows de-interleaved, conv weights reordered to [OC][K][IC],
 * FFN w1/w3 interleaved). compute_type: TSN_COMPUTE_F16 or TSN_COMPUTE_BF16. */
int tsn_dit_load(tsn_device * dev, const char * gguf_path, int compute_type, tsn_dit ** out);
/* Host-only check of a DiT GGUF, no device needed: DitModel::load's geometry keys
 * (src/dit.cpp:29-46) and every tensor the forward reads, present with its expected shape
 * (WeightSet::need, src/net.mm:110-118). TSN_ERR_IO (unreadable), TSN_ERR_FORMAT (bad magic,
 * version, truncated header or tensor table, tensor data past the end of the file;
 * src/gguf.cpp:73-151), TSN_ERR_MISSING (a tensor absent or mis-shaped), TSN_ERR_ARG (geometry
 * this build does not provide). tsn_dit_load fails with the same codes. geom and weight_bytes (the
 * device bytes the weights take) may be null. */
int tsn_dit_inspect(const char * gguf_path, tsn_dit_geom * geom, size_t * weight_bytes);
/* Same model from the seeded synthetic fixture generated on the device: bit-identical to loading
 * the file tsn_gguf_write_synthetic writes for the same geometry and seed. */
int tsn_dit_load_synthetic(tsn_device * dev, const tsn_dit_geom * g, uint64_t seed, int compute_type, tsn_dit ** out);
int tsn_dit_free(tsn_dit * m);
int tsn_dit_get_geom(tsn_dit * m, tsn_dit_geom * out);
size_t tsn_dit_weight_bytes(tsn_dit * m);

/* Fix the sequence geometry and allocate every activation buffer (src/dit.cpp:63-88):
 * T latent rows, clip_S clip rows, text_S text rows. arms = 2 runs one generation's cond and uncond
 * arms batched in one forward (CFG); arms = 2G (4, 6, 8) batches G independent generations, each
 * with its two arms (cond at 2g, uncond at 2g + 1), all stepping on the same schedule; arms = 1
 * runs a single arm (the 2-GPU CFG split). */
int tsn_dit_prepare(tsn_dit * m, uint32_t T, uint32_t clip_S, uint32_t text_S, uint32_t arms);

/* Per-generation conditioning, the outputs of DitModel::prep_conditioning / prep_text_arm
 * (src/dit.cpp:55-192): clip_pp [G][C,H], sync_gather [G][T,H] shared by a generation's arms;
 * text_pp [arms][TS,H] and gcmlp [arms][H] per arm (cond first). Any-pointers; copied in. */
int tsn_dit_set_conditioning(tsn_dit * m, const float * clip_pp, const float * sync_gather,
                             const float * text_pp, const float * gcmlp);
/* Read back the model's conditioning buffers (the layouts of tsn_dit_set_conditioning); any
 * pointer may be null to skip that buffer. */
int tsn_dit_get_conditioning(tsn_dit * m, float * clip_pp, float * sync_gather, float * text_pp, float * gcmlp);
/* DitModel::prep_conditioning (src/dit.cpp:55-135) on the GPU for the prepared geometry:
 * clip_f [C][1024] (C = the prepared clip rows) and sync_f [sync_S][768] f32, host or device
 * pointers. Writes the model's clip_pp and sync_gather and keeps clip_fc for the text arms.
 * Needs the once-per-generation conditioning weights in the model's source (loaded on first use)
 * and H = 1024; one generation (arms 1 or 2). */
int tsn_dit_prep_conditioning(tsn_dit * m, const float * clip_f, const float * sync_f, int sync_S);
/* DitModel::prep_text_arm (src/dit.cpp:137-192) for CFG arm `arm` (< the prepared arms):
 * text_cat [TS][2048] and gtext [1024] f32 -> the model's text_pp[arm] and gcmlp[arm].
 * After tsn_dit_prep_conditioning; together they replace tsn_dit_set_conditioning. */
int tsn_dit_prep_text_arm(tsn_dit * m, int arm, const float * text_cat, const float * gtext);

/* Latent x [G][T,64] (any-pointer in / out). */
int tsn_dit_set_x(tsn_dit * m, const float * x);
int tsn_dit_get_x(tsn_dit * m, float * x_out);

/* DitModel::forward (src/dit_fwd.cpp:104-304) for every arm at once at flow time t; writes
 * flow [arms][T,64] to flow_out (any-pointer). Runs as a replayed CUDA graph. */
int tsn_dit_forward(tsn_dit * m, float t, float * flow_out);
/* The same forward run eagerly, keeping the reference's per-tap tensors (src/dit_fwd.cpp:151-301). */
int tsn_dit_forward_taps(tsn_dit * m, float t, float * flow_out);
/* Copy tap `name` of arm `arm` from the last tsn_dit_forward_taps, in the reference's row-major
 * layout, into out (n floats at most). Returns the tap length through *len. */
int tsn_dit_tap(tsn_dit * m, const char * name, int arm, float * out, size_t n, size_t * len);

/* One sampler step (src/pipeline.cpp:146-148): both forwards + cfg_euler, x updated in place on the
 * device. Requires arms = 2. */
int tsn_dit_step(tsn_dit * m, float t, float cfg, float dt);
/* The Euler loop of src/pipeline.cpp:142-155 (t = 1 - s/steps, dt = t_{s+1} - t_s) over `steps`. */
int tsn_dit_sample(tsn_dit * m, int steps, float cfg);
/* Run `n` more steps of the schedule installed by the last tsn_dit_schedule (for timing loops). */
int tsn_dit_schedule(tsn_dit * m, int steps, float cfg);
int tsn_dit_run_steps(tsn_dit * m, int n);
/* The sampler with the CFG pair split over two GPUs (src/pipeline.cpp:142-155 with the cond and
 * uncond forwards of each step on different devices, arms = 1 on each), as three calls that only
 * issue work on the device's stream (no synchronisation, no host copies, no allocation), so that a
 * caller can capture a whole step, its own flow exchange included (e.g. an NCCL all-gather on the
 * same stream), in one CUDA graph and replay it. Make one eager step before capturing (it loads
 * kernels and creates the library's side streams); tsn_dit_split_schedule then rewinds.
 * tsn_dit_split_schedule: install the t / dt schedule of src/pipeline.cpp:142-145 for `steps` steps
 *   and rewind it to step 0 (synchronises; not for capture).
 * tsn_dit_split_forward: this arm's forward at the schedule's current step; its flow [T,64] f32 is
 *   copied to flow_dev (device memory).
 * tsn_dit_split_update: x += dt_s (fu + cfg (fc - fu)) with fc, fu = flows2_dev[0], flows2_dev[1]
 *   ([2][T,64] f32, device) and the current step's dt (shaders/ops_conv.metal:194-201), then advance
 *   the schedule one step. */
int tsn_dit_split_schedule(tsn_dit * m, int steps);
int tsn_dit_split_forward(tsn_dit * m, float * flow_dev);
int tsn_dit_split_update(tsn_dit * m, const float * flows2_dev, float cfg);
/* End-to-end step through host memory: copy x_host_in to the device, one step, copy x back. */
int tsn_dit_step_host(tsn_dit * m, const float * x_host_in, float * x_host_out, float t, float cfg, float dt);
/* Number of kernels one step (forward + cfg_euler + schedule advance) launches. */
int tsn_dit_kernels_per_step(tsn_dit * m);
/* Per-kernel-class device time of one eagerly launched step, measured with CUDA events around
 * each launch: out[0] tensor-core GEMM ms, out[1] attention ms, out[2] other ms, out[3] GEMM
 * FLOPs, out[4] GEMM launches. */
int tsn_dit_profile_step(tsn_dit * m, double * out5);
/* The same eager forward with one line per launch (name, device ms, TFLOP/s, tile configuration,
 * algorithmic FLOPs) written into out (NUL-terminated, truncated to cap). */
int tsn_dit_profile_ops(tsn_dit * m, char * out, size_t cap);

/* Run the forward up to stamped launch `op` (index in tsn_dit_profile_ops) and that launch once more
 * with per-CTA phase timestamps (globaltimer ns): entry, setup done, first stage landed,
 * accumulator complete, epilogue done, exit, first cluster barrier passed, cluster reduction
 * done (the last two 0 without split-K) — 8 per CTA into out (max_ctas CTAs). adaLN and
 * attention launches stamp entry, upstream wait passed and exit in the first 3 of the 8. */
int tsn_dit_trace_op(tsn_dit * m, int op, unsigned long long * out, size_t max_ctas, int * n_ctas);

/* Run one forward eagerly on the graph's streams with every GEMM, adaLN and attention launch
 * stamping its CTAs (globaltimer ns). Per stamped launch, 5 doubles into out (max_rows rows): op
 * index (as in tsn_dit_profile_ops), earliest CTA entry, earliest start of work (GEMM: first operand
 * stage landed; others: upstream wait passed), latest exit, median exit — in ns from the earliest
 * entry. n_rows receives the number of stamped launches. */
int tsn_dit_timeline(tsn_dit * m, double * out, size_t max_rows, int * n_rows);

/* Time every valid tile configuration (tile width, cluster split-K factor) of each distinct GEMM
 * shape of the prepared forward on this device and keep the fastest (the default is a static cost
 * model). Results stay bit-identical between calls of this model; two processes that tune
 * differently may differ in the last bits. Writes one line per shape into report. */
int tsn_dit_autotune(tsn_dit * m, char * report, size_t cap);

/* The tile of every GEMM launch of the planned forward, 3 ints each into out (max_gemms entries):
 * GEMM index, tile width (2000 + NT for the CTA-pair kernel with NT-token tiles) and K slices (the
 * cluster size, or the partial-tile count of the deepest member of a grouped launch). n_gemms
 * receives the count. Saving this table after tsn_dit_autotune and passing it to
 * tsn_dit_set_tiles later reproduces the tuned forward without re-timing. */
int tsn_dit_get_tiles(tsn_dit * m, int * out, int max_gemms, int * n_gemms);

/* Pin GEMM tiles (n triples as tsn_dit_get_tiles writes them) and re-plan the forward; GEMMs not
 * listed, and entries that do not fit their GEMM, fall back to the static cost model. */
int tsn_dit_set_tiles(tsn_dit * m, const int * tiles, int n);

/* ------------------------------------------------------------------ VAE decoder */
/* VaeModel::decode (src/vae.cpp:17-86) on the GPU: latent [T, latent_dim] f32 -> interleaved audio
 * [T * 2048, out_channels] f32. The f32 weights are held as f16 hi + lo halves (split-weight
 * tcgen05 GEMMs); transposed convs run as polyphase stride-1 convs. */
typedef struct tsn_vae tsn_vae;
/* Load from a VAE GGUF (the tensor names of src/vae.cpp; f32, f16 or bf16 values). */
int tsn_vae_load(tsn_device * dev, const char * gguf_path, tsn_vae ** out);
/* The seeded synthetic VAE (the values tsn_gguf_write_synthetic_vae writes), generated in memory. */
int tsn_vae_load_synthetic(tsn_device * dev, uint32_t latent_dim, uint32_t channels, uint32_t out_channels, uint64_t seed,
                           tsn_vae ** out);
/* Decode latent [T, latent_dim] into audio [T_audio, out_channels] (host or device pointers;
 * audio_cap in floats). The first decode of a length plans and captures its graph. */
int tsn_vae_decode(tsn_vae * v, const float * latent, uint32_t T, float * audio, size_t audio_cap, uint32_t * T_audio);
/* Device time of the last decode (ms, graph only) and the algorithmic FLOPs (2·M·N·K over every
 * conv) of the prepared length. */
double tsn_vae_last_ms(tsn_vae * v);
/* The last decoded length once more, launch by launch, one line per launch (name, device ms). */
int tsn_vae_profile_ops(tsn_vae * v, char * out, size_t cap);
double tsn_vae_flops(tsn_vae * v);
/* Kernel launches in one decode graph of the prepared length. */
int tsn_vae_launches(tsn_vae * v);
int tsn_vae_free(tsn_vae * v);

/* ------------------------------------------------------------------ text encoders */
/* T5Model (src/t5.cpp, src/models.h:40-52) and ClipModel (src/clip.cpp, src/models.h:24-38) on the
 * GPU, one handle type for both. Loading follows WeightSet::load with keep_f32 (src/net.mm:126-173):
 * f32 tensors stay f32 (split-weight GEMMs), others (the T5 file's Q8_0) become f16 by the
 * reference's rounding rule. Returns TSN_ERR_UNSUPPORTED unless the head size is 64. */
typedef struct tsn_encoder tsn_encoder;
/* Replaces T5Model::load (src/t5.cpp:22-59): KV keys t5.* with the reference's defaults. */
int tsn_t5_load(tsn_device * dev, const char * gguf_path, tsn_encoder ** out);
/* Replaces ClipModel::load (src/clip.cpp:6-28): KV keys clip.*. */
int tsn_clip_load(tsn_device * dev, const char * gguf_path, tsn_encoder ** out);
/* Width (d_model / hidden), context (77) and layer count. */
int tsn_encoder_info(tsn_encoder * e, uint32_t * width, uint32_t * ctx, uint32_t * layers);
/* Replaces T5Model::encode (src/t5.cpp:84-131) and ClipModel::encode (src/clip.cpp:30-101): n_ids
 * must equal ctx (ids already padded, as the tokenizers return them); every id must lie inside the
 * vocabulary (TSN_ERR_ARG otherwise; the reference would read past its table). per_token [ctx, width]
 * f32; pooled [width] (CLIP's text_proj of the EOT row; ignored for T5, may be null). Host or device
 * pointers. One CUDA graph per encoder. */
int tsn_encoder_encode(tsn_encoder * e, const int32_t * ids, uint32_t n_ids, float * per_token, size_t per_token_cap,
                       float * pooled, size_t pooled_cap);
/* Device time of the last encode (ms), its algorithmic FLOPs and the weight bytes it streams. */
double tsn_encoder_last_ms(tsn_encoder * e);
double tsn_encoder_flops(tsn_encoder * e);
/* Kernel launches in one encode graph. */
int tsn_encoder_launches(tsn_encoder * e);
double tsn_encoder_weight_bytes(tsn_encoder * e);
/* The encode's launches once more eagerly, one line per launch (name, device ms). */
int tsn_encoder_profile_ops(tsn_encoder * e, char * out, size_t cap);
int tsn_encoder_free(tsn_encoder * e);

/* ------------------------------------------------------------------ transformer-block operators */
/* Three operators of a transformer block, without counterpart in the reference. They follow one another
 * inside a block: norms around a branch (tsn_block_norm), rotary positions of its queries and keys
 * (tsn_rope_axes), differential attention (tsn_diff_attn). Each issues one kernel on the device's
 * stream and returns without synchronising; a size of zero rows is no work and no error. Inputs and
 * results are device memory that the caller owns; results may not overlap inputs except where a call
 * says so. All sums, softmax statistics and norms are held in 32 bits; a result is rounded once. */
enum { TSN_F32 = 0, TSN_F16 = 1, TSN_BF16 = 2 };
enum { TSN_NORM_NONE = 0, TSN_NORM_RMS = 1, TSN_NORM_LAYER = 2 };

/* Rows of C consecutive elements: row t of batch b starts at element b * sb + t * st of p. A stride of
 * 0 repeats the row (inputs only), so one row per batch has st = 0. p null: the term is absent. */
typedef struct tsn_rows { void * p; int64_t sb, st; } tsn_rows;
/* Head rows of consecutive elements: token s, head h of batch b starts at element b*sb + s*ss + h*sh. */
typedef struct tsn_heads { void * p; int64_t sb, ss, sh; } tsn_heads;

/* Norms before and after a block, fused with the block's gate and residual scale. Per row of C:
 *   x_out = r * x + act(gate) * Npost(y)          h = Npre(x_out) * (1 + scale) + shift
 * RMS: N(u) = u / sqrt(mean(u^2) + eps) * w (+ b); LAYER: N(u) = (u - mean) / sqrt(var + eps) * w (+ b);
 * NONE: N(u) = u. r is res_vec [C] where given, else res_scale; act is tanh if gate_tanh, to 2^-20 of its value. Npre sees
 * x_out before it is rounded to xtype. Absent terms: y (then x_out = r * x), gate (1), scale (0), shift
 * (0), weights (1), biases (0); x_out or h may be absent, not both. x and x_out are of xtype, which
 * is `type` or TSN_F32; y, h, gate, shift and scale are of `type`; weights, biases and res_vec are f32.
 * x_out may be x, and h may be y, at the same strides. C 1..16384; any strides and alignment (rows that
 * all start at 16-byte boundaries are read 16 bytes at a time, at pairs of elements a pair at a time). */
typedef struct tsn_block_norm_args {
    uint32_t B, T, C;
    int32_t xtype, type, post, pre, gate_tanh;
    float post_eps, pre_eps, res_scale;
    tsn_rows x, y, x_out, h, gate, shift, scale;
    const float * post_w, * post_b, * pre_w, * pre_b, * res_vec;
} tsn_block_norm_args;
int tsn_block_norm(tsn_device * dev, const tsn_block_norm_args * a);

/* Rotary positions with 1 to 4 axes (time, height, width, ...), after an optional RMSNorm of each head.
 * A head of D elements has P = sum(pairs) rotated pairs, pairs[0] of the first axis, then pairs[1] of
 * the second, and so on; elements from 2 P on pass through. Pair i of the n pairs of axis a turns by
 * pos[a] * scale[a] * theta[a]^(-i / n): (u, v) -> (u cos - v sin, u sin + v cos). The pair's
 * elements are 2 j, 2 j + 1 (TSN_ROPE_INTERLEAVED) or j, j + P (TSN_ROPE_HALF), j counting over all axes.
 * tsn_rope_plan fills the plan (host only, no device): each pair's turns per position as a 64-bit
 * fraction, so that an angle keeps its full precision at any 32-bit position. */
enum { TSN_ROPE_INTERLEAVED = 0, TSN_ROPE_HALF = 1 };
enum { TSN_ROPE_MAX_PAIRS = 128, TSN_ROPE_MAX_AXES = 4 };
typedef struct tsn_rope_plan_t {
    uint32_t D, axes, P;
    int32_t layout;
    uint64_t turn[TSN_ROPE_MAX_PAIRS];
    uint8_t axis[TSN_ROPE_MAX_PAIRS];
} tsn_rope_plan_t;
/* D even, 2..256, 2 P <= D; theta > 0, scale and the turns that they give finite. */
int tsn_rope_plan(uint32_t D, uint32_t axes, const uint32_t * pairs, const double * theta, const double * scale,
                  int layout, tsn_rope_plan_t * out);
/* q [B, S, Hq, D] and k [B, S, Hk, D] of `type` into q_out and k_out (the inputs themselves, at the same
 * strides, or other memory, e.g. a cache). Either pair may be absent (p null). pos: int32, axis a of
 * token s of batch b at pos[b * pos_sb + s * pos_ss + a] (pos_sb 0: shared by the batch). q_norm, k_norm:
 * f32 [D] weights of the heads' RMSNorm, or null for none. */
typedef struct tsn_rope_args {
    uint32_t B, S, Hq, Hk;
    int32_t type;
    float eps;
    tsn_heads q, k, q_out, k_out;
    const int32_t * pos;
    int64_t pos_sb, pos_ss;
    const float * q_norm, * k_norm;
} tsn_rope_args;
int tsn_rope_axes(tsn_device * dev, const tsn_rope_plan_t * plan, const tsn_rope_args * a);

/* Differential attention: the difference of two softmax maps over shared values, then an RMSNorm of each
 * head. A query or key head is [q1 | q2] of d elements each, a value head has 2 d:
 *   A_m = softmax(scale * q_m k_m^T) over the visible keys,  o = (A_1 - lambda A_2) v
 *   lambda = exp(lq1 . lk1) - exp(lq2 . lk2) + lambda_init
 *   out = o / sqrt(mean(o^2) + eps) * norm_w * (1 - lambda_init)
 * q [B, Sq, H, 2 d], k and v [B, Sk, Hk, 2 d] (query head h reads kv head h / (H / Hk)), out as q, all of
 * `type` TSN_F16 or TSN_BF16; d is 32 or 64, H / Hk at most 128. Base addresses and strides of q, k, v and
 * out are multiples of 16 bytes; those of k and v are positive, or 0 for the batch in both (shared keys).
 * scale 0 means 1 / sqrt(d).
 * Visible keys of query i in batch b, with n = key_len[b] (int32, clamped to 0..Sk; null: Sk): j < n; and
 * key_mask[b * mask_sb + j] != 0 (bytes; null: all); and with causal j <= i + n - Sq, so the last query
 * sees the last key. A row that sees no key is zero, whatever eps is. What masked keys and values hold has no effect, NaN
 * and infinities included; a row that sees a non-finite value, or has a score that is NaN or +infinity, is NaN; a key
 * whose score is -infinity has no share in that map.
 * lq1 .. lk2: f32 vectors of d, one per query head lam_sh elements apart (0: shared). norm_w: f32 [2 d] or
 * null for ones.
 * The probabilities are rounded to `type` before the product with v, as the tensor cores take them, and their sum is
 * that of the rounded ones.
 * Few query rows over many keys split the keys over several CTAs, whose sums meet in a workspace. Calls take turns at
 * the device handle's (32 MiB, allocated at its first such call and kept), whatever streams they are on. A call captured
 * in a CUDA graph has one of its own size that belongs to the graph, so replays may run beside one another and beside
 * other calls; executables made from one graph share it, as they share the results. A graph is replayed while the handle
 * is there (its error word is the handle's). At most 2^30 queries, keys and query rows of a kv
 * head (Sq * H / Hk), 65535 sequences and heads. */
typedef struct tsn_diff_attn_args {
    uint32_t B, Sq, Sk, H, Hk, d;
    int32_t type, causal;
    float scale, lambda_init, eps;
    tsn_heads q, k, v, out;
    const int32_t * key_len;
    const uint8_t * key_mask;
    int64_t mask_sb;
    const float * lq1, * lk1, * lq2, * lk2;
    int64_t lam_sh;
    const float * norm_w;
} tsn_diff_attn_args;
int tsn_diff_attn(tsn_device * dev, const tsn_diff_attn_args * a);

/* ---- a key/value cache in pages that many sequences share: appending to it, attention over it.
 * B sequences. The cache is P pages of `page` tokens each (a power of two, 16..1024) of Hk heads of D elements, keys in k and
 * values in v: slot t of page p, head h starts at element p * sb + t * ss + h * sh, any order of the three. Place j of
 * sequence b (its j-th token) lies in page table[b * table_sb + j / page], slot j % page; M entries a sequence. An entry
 * outside 0..P - 1 is no page: what would be written there is dropped, and its keys are not seen.
 * A call brings N rows of new tokens. Those of sequence b are rows q_start[b] .. q_start[b + 1] - 1 (q_start: B + 1 ascending
 * numbers, 0..N; null: N = B, row b). len[b] counts the sequence's tokens in the cache, the new ones included: the i-th
 * of n new tokens has place len[b] - n + i. Places below 0 or from M * page on are in no page. Rows that belong
 * to no sequence are left as they were. table, len and q_start are int32 and read on the device; whatever they hold, nothing
 * outside the pages is touched. Sequences may share pages that a call only reads.
 * k and v are of `type`, TSN_F16 or TSN_BF16; base addresses and strides are multiples of 16 bytes, strides positive. At most
 * 65535 sequences and heads, 2^30 new tokens and places of a sequence, 2^31 - 1 pages. */
typedef struct tsn_paged {
    uint32_t B, N, P, M, page, Hk, D;
    int32_t type;
    tsn_heads k, v;
    const int32_t * table;
    int64_t table_sb;
    const int32_t * len, * q_start;
} tsn_paged;

/* Appends new tokens: an optional RMSNorm and the rotary positions of `plan` for queries and keys, as tsn_rope_axes does it, keys
 * and values into their pages. q [N, Hq, D] into q_out (Hq 0 or q.p null: keys and values only), k and v [N, Hk, D]: row i,
 * head h starts at element i * sb + h * st. q, k and v are of xtype, which is c.type or TSN_F32; q_out is of c.type, and may be
 * q at the same strides where the types agree. D is a multiple of 8, 8..256; addresses and strides are multiples of 16 bytes.
 * pos: int32, axis a of row i at pos[i * pos_ss + a]; null: the token's place (plans of one axis).
 * means (or p null): of c.type, page p, head h at element p * sb + h * st: the mean over the keys that the page holds of its
 * sequence, as they are stored, for every page that a new token went into. Sequences that share a page
 * they write to, or a row of means, leave it undefined. */
typedef struct tsn_cache_append_args {
    tsn_paged c;
    uint32_t Hq;
    int32_t xtype;
    float eps;
    tsn_rows q, k, v, q_out, means;
    const int32_t * pos;
    int64_t pos_ss;
    const float * q_norm, * k_norm;
} tsn_cache_append_args;
int tsn_cache_append(tsn_device * dev, const tsn_rope_plan_t * plan, const tsn_cache_append_args * a);

/* Attention of the new tokens over their sequences' caches (appended before): out = softmax(scale q k^T) v over the visible keys.
 * q and out [N, H, D] of c.type, row i, head h at element i * sb + h * st; query head h reads kv head h / (H / Hk), H / Hk at
 * most 128; D is 64 or 128. scale 0 means 1 / sqrt(D). A token at place p sees place j of its sequence where j < len[b];
 * with causal j <= p; and with window > 0 (causal only) j > p - window. A row that sees no key is zero.
 * What unseen keys and values hold has no effect, NaN and infinities included. Of seen ones: a row with a score of NaN or +infinity is
 * NaN; a key whose score is -infinity has no share, and a row that sees no others is zero; a value that is not finite makes its
 * column of the row so, NaN or an infinity, however small its key's share (which of them is left open: 0 times infinity is NaN where the
 * product takes it, but where the rows of a tile see different keys such values are added apart).
 * The probabilities are rounded to `type` before the product with v, as the tensor cores take them, and the sum that divides is of the
 * rounded ones. In f16, keys whose share is below 2^-21 of the greatest one's lose bits of it: each is off by at most 2^-32 of that.
 * most: new tokens of a sequence at most, as far as the caller knows (0: not known); it decides which kernel
 * runs, never the result's extent. Split keys meet in a workspace, as those of tsn_diff_attn do. */
typedef struct tsn_paged_attn_args {
    tsn_paged c;
    uint32_t H, most;
    int32_t causal;
    uint32_t window;
    float scale;
    tsn_rows q, out;
} tsn_paged_attn_args;
int tsn_paged_attn(tsn_device * dev, const tsn_paged_attn_args * a);
/* A test hook for the failure path: the call by its kernel for few rows, in which the waits of block `block` for its first loads
 * count as run out (nothing hangs, the loads land). Expected result: TSN_ERR_TIMEOUT where there is such a block with keys to read;
 * out is undefined then, and later calls are not affected. Synchronises. */
int tsn_selftest_paged_timeout(tsn_device * dev, const tsn_paged_attn_args * a, uint32_t block);

/* Causal attention over `picks` pages of the cache, chosen for each new token and kv head by a cheap score: page x scores
 * (sum of the group's query heads) . means[x], in 64 bits. For a token at place p, with its own page o = p / page, the
 * candidates are pages 0..o; pages below `first` and above o - last (the token's own among them; last at least 1) come before
 * all others, then higher scores, and of equal scores the lower page. chosen [N, Hk, picks], int32: the chosen pages in
 * ascending order, then -1 where there are fewer. out as tsn_paged_attn with causal over the keys of the chosen pages. means is
 * what tsn_cache_append keeps, all finite; entries of the table that are no page score as zero means do. A token at a place
 * below 0 or from M * page on chooses nothing and gets zeros. first + last <= picks <= 1024; M at most 16384. */
typedef struct tsn_sparse_attn_args {
    tsn_paged c;
    uint32_t H, picks, first, last;
    float scale;
    tsn_rows q, out, means;
    int32_t * chosen;
} tsn_sparse_attn_args;
int tsn_sparse_attn(tsn_device * dev, const tsn_sparse_attn_args * a);

/* For a Python binding of the operators on tensors: a call whose tensors have the form of the call before (shape,
 * strides, type, place) needs no checks, only their addresses. `view` is the function of the tensor type's DLPack
 * exchange table that describes an object as a DLTensor, `item` the interpreter's PyTuple_GetItem, `type` the objects'
 * exact type, `none` the None object. tsn_form_take takes a tuple of n objects, writes their addresses (null for
 * None) to *to[i] and returns 1 if every one has
 * the recorded form, or, with `record`, records the forms. Otherwise it returns 0, what lies at *to[i] is undefined,
 * and nothing is recorded any more. The caller holds the interpreter's lock. Host only. */
enum { TSN_FORM_TENSORS = 11 };
typedef struct tsn_form_tensor {
    int32_t there, device_type, device, ndim;
    uint32_t dtype;
    int64_t shape[4], strides[4];
} tsn_form_tensor;
typedef struct tsn_form {
    int (*view)(void * object, void * dl_tensor);
    void * (*item)(void * tuple, intptr_t i);
    void * type, * none;
    uint32_t n, valid;
    void ** to[TSN_FORM_TENSORS];
    tsn_form_tensor t[TSN_FORM_TENSORS];
} tsn_form;
int tsn_form_take(tsn_form * f, int record, void * tuple);

/* ------------------------------------------------------------------ fixtures */
/* Write the seeded synthetic DiT GGUF (with_prep adds the conditioning-prep tensors). Host only. */
int tsn_gguf_write_synthetic(const char * path, const tsn_dit_geom * g, uint64_t seed, int with_prep);
/* Write the seeded synthetic VAE decoder GGUF (f32 tensors: conv k7 latent_dim -> 16 channels,
 * five upsampling blocks at strides 8, 8, 4, 4, 2 with widths 8, 4, 2, 1, 1 x channels, final conv
 * to out_channels; tensor names of src/vae.cpp). Host only. */
int tsn_gguf_write_synthetic_vae(const char * path, uint32_t latent_dim, uint32_t channels, uint32_t out_channels,
                                 uint64_t seed);
/* Write the seeded synthetic T5 encoder GGUF (Q8_0 matrices and embedding, f32 norms and relative
 * bias; tensor names and KV keys of src/t5.cpp; vocabulary 32128). Host only. */
int tsn_gguf_write_synthetic_t5(const char * path, uint32_t d_model, uint32_t d_ff, uint32_t layers, uint32_t heads,
                                uint64_t seed);
/* Write the seeded synthetic MetaCLIP text encoder GGUF (f32; names and keys of src/clip.cpp;
 * vocabulary 49408, context 77). Host only. */
int tsn_gguf_write_synthetic_clip(const char * path, uint32_t hidden, uint32_t layers, uint32_t heads, uint64_t seed);

#ifdef __cplusplus
}
#endif

#endif /* TSN_H */
