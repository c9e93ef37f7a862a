/*
 * cutdet.h -- C ABI of libcutdet.so, the MI355X (gfx950) classify+segment hot path.
 *
 * The reference (play4honor/Cut-Detection) is pure Python and has no FFI of its own; each entry
 * point below names the Python call it stands in for.  Bindings use plain pointers and sizes
 * (ctypes: cut-detection_amd/cutdet/_lib.py).
 *
 * Conventions
 *   - every function returns 0 on success and a negative CD_E* code on failure; the message for
 *     the calling thread's last failure is cd_last_error().  Nothing throws across the ABI.
 *   - `stream` is a hipStream_t passed as void* (NULL = the default stream).  All work is queued
 *     on it.  Steady-state calls do not synchronise; a call that has to grow the workspace or sees
 *     a new source geometry (other H0 x W0 -> net_h x net_w) synchronises the stream once while it
 *     re-allocates / uploads its resize tables (cd_reserve() and a first warm-up call avoid both).
 *   - pointers marked "device" must be device memory on the handle's GPU.  Frames, activations
 *     and results are caller-owned; the handle owns the packed weights and an activation
 *     workspace that grows only inside cd_reserve()/the first call that needs more.
 *   - a handle is bound to one device and is not thread-safe; distinct handles are independent.
 *     Use one stream per handle at a time: consecutive calls on different streams are not ordered
 *     against each other by the library (the activation workspace is shared by all of them).
 *
 * What is pinned against the reference and what is not
 *   - fp32 forward, max/argmax, run-length tables, glue/merge and CSV are checked against outputs of
 *     the reference itself (logits to 1e-3, everything else exact, the per-segment means included:
 *     for segments shorter than 32768 frames cd_rle adds the maxima in the order of torch's CPU
 *     float32 sum kernel, so the mean - which decides the order in which orphans are glued - is the
 *     reference's torch.mean bit for bit.  From 32768 elements on torch splits a reduction over its
 *     threads and the reference's own value depends on the machine; there the mean is the fp64 sum
 *     rounded once).
 *   - the resize for geometries other than an odd integer scale (a pure point sample such as
 *     1280x720 -> 256x144) restates OpenCV's published 8-bit INTER_LINEAR arithmetic without an
 *     OpenCV build to compare with: parity unpinned.
 *   - CD_BF16 has no counterpart in the reference: parity unpinned; its logits are within 4.2e-2 of
 *     the fp32 result on the test clips.
 */
#ifndef CUTDET_H
#define CUTDET_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct cd_handle cd_handle;

enum {
    CD_OK = 0,
    CD_EINVAL = -1,   /* bad argument / unsupported shape */
    CD_EHIP = -2,     /* a HIP runtime call failed */
    CD_ECAP = -3,     /* caller-provided capacity too small */
    CD_ENOMEM = -4
};

/* pipeline stages, for cd_timing_read() */
enum {
    CD_STAGE_PREPROCESS = 0,
    CD_STAGE_CONV1 = 1,      /* block 1 (with the fused resize when called through cd_forward_u8) */
    CD_STAGE_CONV2 = 2,      /* block 2: 60 % of the network's FLOPs */
    CD_STAGE_CONV3_HEAD = 3, /* block 3 + pooling + both linear layers + max/argmax */
    CD_STAGE_RLE = 4,        /* the four run-length kernels of one cd_rle call */
    CD_STAGE_COUNT = 5
};

/* Arithmetic type of the forward pass.  CD_F32: everything in fp32 (what the reference computes): exact
 * products accumulated in fp32.  Blocks 2 and 3 and the head use the fp32 matrix instructions; block 1 of u8
 * frames gets the same exact products from the bf16 matrix cores - a byte is exact in bfloat16 and the fp32
 * weight is written as three bfloat16 terms that sum to it exactly - unless CD_OPT_F32_BLOCK1_FP32_MFMA
 * (cd_set_option) asks for the fp32 instructions there too.
 * CD_BF16: the three convolutions multiply bfloat16 inputs/activations and weights on the bf16
 * matrix cores with fp32 accumulation; bias, pooling/affine epilogues and the head stay fp32.
 * Logits then differ from the fp32 result by a few 1e-2; class ids are unchanged on inputs with
 * clear margins.
 * CD_BF16_SPLIT: blocks 2 and 3 multiply fp32 values split into two bfloat16 terms each
 * (v = hi + lo to 2^-17) on the bf16 matrix cores, all four partial products, fp32 accumulation.
 * Block 1 on u8 frames also runs on the bf16 matrix cores: a byte is exact in bfloat16, and the
 * weights carry the 1/255 as hi + lo terms (block 1 on float frames, cd_forward, is fp32).
 * Epilogues and head are fp32.  Logits stay within 1e-3 of the fp32 result (measured: a few 1e-5
 * on the test clips). */
enum { CD_F32 = 0, CD_BF16 = 1, CD_BF16_SPLIT = 2 };
enum { CD_BGR = 0, CD_RGB = 1 };         /* channel order of u8 frames in memory */

int cd_version(void);
const char* cd_last_error(void);

/* Builds the classifier from a weight blob (format: cut-detection_amd/cutdet/weights.py).
 * Replaces frameID/net.py:193-217 load_and_glue_nets() + segment_video.py:33-34 eval()/to(device). */
int cd_create(cd_handle** out, const void* weights_blob, size_t nbytes, int device, int dtype);
void cd_destroy(cd_handle* h);

/* Sizes the activation workspace for batches of up to max_frames frames of network input
 * height net_h (width is always 256).  Optional: the forward calls grow it on demand.  Returns
 * with the workspace ready (its zeroing has completed), whatever stream the next call uses. */
int cd_reserve(cd_handle* h, int max_frames, int net_h);

/* Resize + normalise n decoded frames.
 * Replaces frameID/data.py:218-228 (cv2.resize INTER_LINEAR to w x h, float32, HWC->CHW,
 * BGR->RGB, /255).  src: device u8 [n][H0][row_stride bytes], pixels interleaved 3 bytes;
 * frame_stride = bytes between frames.  dst: device f32 [n][3][h][w], RGB planes in [0,1]. */
int cd_preprocess(cd_handle* h, const uint8_t* src, int n, int H0, int W0,
                  int64_t row_stride, int64_t frame_stride, int chan_order,
                  float* dst, int net_h, int net_w, void* stream);

/* The resize alone, u8 in, u8 out.
 * Replaces cv2.resize(frame, (net_w, net_h), INTER_LINEAR) at frameID/data.py:220-222 by itself.
 * src as in cd_preprocess; dst: device u8 [n][net_h][net_w][3], pixels interleaved in the source's
 * channel order.  Its output fed to cd_forward_u8 (as net_h x net_w frames) gives the bits of
 * cd_forward_u8 on the source frames: a caller with the next batch at hand can run this resize on a
 * second stream while the previous batch is being classified (memory-bound work beside matrix-bound
 * work), which the single fused call cannot.  Keeps its own resize tables, so alternating it with
 * forward calls of another geometry does not re-upload anything. */
int cd_resize_u8(cd_handle* h, const uint8_t* src, int n, int H0, int W0,
                 int64_t row_stride, int64_t frame_stride,
                 uint8_t* dst, int net_h, int net_w, void* stream);

/* NV12 frames (what hardware video decoders deliver: a luma plane, then a half-height plane of
 * interleaved U,V pairs, each pair shared by a 2x2 pixel block) -> interleaved 3-byte pixels, the
 * input format of cd_preprocess / cd_forward_u8.  Stands in for the colour conversion that
 * cv2.VideoCapture.read() has already applied to the frames the reference sees
 * (frameID/data.py:213); BT.601 limited range in the 20-bit fixed point OpenCV's
 * cvtColor(COLOR_YUV2BGR_NV12) publishes.  Parity unpinned: the reference never handles NV12.
 * y: device u8, n planes of rows of y_row_stride bytes, y_frame_stride bytes apart; uv likewise.
 * Output row r of a frame is built from luma row y_rows[r] and chroma row uv_rows[r] (device
 * int32 [n_rows] each; NULL = row r and row y_row/2), so a caller that uploaded only the rows the
 * resize samples converts just those.  dst: device u8 [n][n_rows][W0][3].  W0 must be even. */
int cd_nv12_to_bgr(cd_handle* h, const uint8_t* y, const uint8_t* uv, int n, int W0,
                   int64_t y_row_stride, int64_t uv_row_stride,
                   int64_t y_frame_stride, int64_t uv_frame_stride,
                   const int32_t* y_rows, const int32_t* uv_rows, int n_rows,
                   uint8_t* dst, int chan_order, void* stream);

/* prod_net forward on preprocessed frames.
 * Replaces net(batch) at segment_video.py:45 (frameID/net.py:33-40,62-68,122-133) and, through
 * maxv/argmax, torch.max(scores, 1) at frameID/segmentation.py:37.
 * x: device f32 [n][3][net_h][256], net_h in 27..215 (the three 3x3 poolings must leave a row;
 * above 215 the block-2 activation of one frame no longer fits a CU's LDS).  logits: device
 * f32 [n][3].  maxv (f32 [n]) and argmax (i64 [n]) may each be NULL.  Ties resolve to the lowest
 * class index.  The max-pooling ignores a NaN among finite inputs where torch would propagate
 * it; decoded u8 frames cannot produce one. */
int cd_forward(cd_handle* h, const float* x, int n, int net_h, int net_w,
               float* logits, float* maxv, int64_t* argmax, void* stream);

/* cd_preprocess + cd_forward fused: the resized frame never reaches HBM.
 * Replaces the data.py:218-228 -> segment_video.py:44-45 chain for one batch.
 * Every row of every frame must be readable for its full row_stride bytes (the last row of the last
 * frame included): when row_stride is a multiple of 16 the general resize fetches rows in 16-byte
 * pieces and may read up to 15 bytes past a row's W0*3 pixel bytes, never past row_stride. */
int cd_forward_u8(cd_handle* h, const uint8_t* src, int n, int H0, int W0,
                  int64_t row_stride, int64_t frame_stride, int chan_order,
                  int net_h, int net_w,
                  float* logits, float* maxv, int64_t* argmax, void* stream);

/* The reference's whole hot loop in one call: n decoded frames resident in device memory, classified
 * in batches of `batch` frames.  Replaces segment_video.py:42-58 (`for batch in dl: yy.append(
 * net(batch))`) together with the data.py:218-228 preprocessing of every frame.  src, strides,
 * chan_order, net_h, net_w as in cd_forward_u8; logits [n][3], maxv [n], argmax [n] (the last two may
 * be NULL) are written at the frames' own rows.  Results are bit-identical to calling cd_forward_u8
 * batch by batch.  What the single-batch call cannot do: consecutive batches alternate between two
 * activation workspaces, the caller's stream and a side stream, so the start-up, tail and
 * per-frame serial phases of one batch's kernels fill with the other batch's work; and for source
 * geometries that need a real resize (not a point sample) the resize of the batches ahead runs as a
 * separate memory-bound pass on a third stream beside the matrix-bound classification.  The call
 * forks from and joins back into `stream`: everything it queued is ordered before whatever the
 * caller queues on `stream` afterwards, and it does not synchronise in the steady state (first use
 * creates the second workspace).  The two side streams exist once per device and are shared by every
 * handle on it (a process has few hardware queues; a pair per handle would put streams of one call on
 * the same queue): range calls of different handles that overlap in time on one device stay correct,
 * their side-stream work is queued one call behind the other.  n <= batch is exactly cd_forward_u8. */
int cd_forward_u8_range(cd_handle* h, const uint8_t* src, int64_t n, int batch, int H0, int W0,
                        int64_t row_stride, int64_t frame_stride, int chan_order,
                        int net_h, int net_w,
                        float* logits, float* maxv, int64_t* argmax, void* stream);

/* How cd_forward_u8_range schedules its work; every setting but the last gives the same bits.  No counterpart in the
 * reference.  The defaults can also be set through the environment when a handle is created
 * (CUTDET_RANGE_MODE, CUTDET_FUSED12, CUTDET_RANGE_ONE_STREAM, CUTDET_S2_TWO_WAVES, CUTDET_RESIZE_ROWS,
 * CUTDET_F32_BLOCK1_FP32_MFMA = 0 or 1).  CD_OPT_SPLIT_TWO_WAVES, CD_OPT_RESIZE_ROWS and CD_OPT_F32_BLOCK1_FP32_MFMA apply to every entry point that runs those kernels, not
 * only to the range call.
 *   CD_OPT_RANGE_BY_STAGE   0 (default): whole batches alternate between the two streams.  1: block 1
 *                           of every batch on one stream, blocks 2 + 3 on the other.
 *   CD_OPT_FUSE_BLOCKS12    CD_BF16_SPLIT handles only.  1: the resize pass writes the first block's
 *                           bfloat16 operand cells and blocks 1 + 2 run as ONE kernel whose block-1
 *                           activations stay in LDS (no 835 KB per frame written to and read back from
 *                           HBM).  0 (default): separate kernels, which is the faster of the two on the
 *                           measured geometries - the fused kernel fills every CU's registers and LDS,
 *                           so nothing overlaps with it.
 *   CD_OPT_RANGE_ONE_STREAM 1: everything on the caller's stream (for measurements: per-stage event
 *                           times are then the kernels' own durations).
 *   CD_OPT_SPLIT_TWO_WAVES  CD_BF16_SPLIT handles only.  1: block 2 runs two waves per SIMD (256 registers
 *                           and one patch buffer each).  0 (default): one wave per SIMD with double-buffered
 *                           patches, the faster of the two on the measured geometries (the two-wave
 *                           kernel waits for its weights, which a second wave's traffic delays in L2).
 *   CD_OPT_RESIZE_ROWS      The stand-alone resize (cd_resize_u8, and the resize pass of the range call).
 *                           0 (default): one thread per output pixel reads its taps from global memory; no
 *                           LDS, so its workgroups find room on a CU beside the convolution kernels'.
 *                           1: one workgroup per output row stages the two source rows in LDS (needs
 *                           16-byte aligned rows; used anyway when the default kernel does not apply: output
 *                           widths that are not a multiple of 4, rows shorter than 8 bytes).
 *   CD_OPT_F32_BLOCK1_FP32_MFMA  CD_F32 handles, u8 sources.  0 (default): block 1 multiplies the frame's bytes (exact in
 *                           bfloat16) with the fp32 weights written as three bfloat16 terms (hi + lo + lo2 == w
 *                           exactly) on v_mfma_f32_16x16x32_bf16: exact products, fp32 accumulation - what the fp32
 *                           matrix instructions compute, in another order of additions and a third of the time.
 *                           1: block 1 on v_mfma_f32_16x16x4_f32 as well.  This option changes low-order bits of
 *                           the logits (both settings agree with the reference to < 1e-5); cd_forward (float
 *                           frames) always uses the fp32 instructions. */
enum { CD_OPT_RANGE_BY_STAGE = 0, CD_OPT_FUSE_BLOCKS12 = 1, CD_OPT_RANGE_ONE_STREAM = 2, CD_OPT_SPLIT_TWO_WAVES = 3,
       CD_OPT_RESIZE_ROWS = 4, CD_OPT_F32_BLOCK1_FP32_MFMA = 5, CD_OPT_COUNT = 6 };
int cd_set_option(cd_handle* h, int option, int value);

/* cd_forward_u8 for callers that cannot allocate device memory (code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc).  No counterpart in the reference.  Same arguments
 * and results as cd_forward_u8 (bit-identical), but the activations between the blocks live in a
 * fixed 32 MiB array in the library's device image instead of the handle's workspace, and the call
 * allocates and frees nothing and records no timing events.  Limit: the batch must fit that array -
 * 34 frames at a network input height of 144 rows (more at smaller heights); a larger batch returns
 * CD_ECAP.  Every call on a GPU shares that GPU's array: calls that overlap on one GPU (other
 * streams, other handles, other threads) race.  The first call on a device, and the first after the
 * input height or the activation cell size changed (CD_BF16 handles store 2-byte cells, the others
 * 4-byte ones), clears the array and synchronises `stream` once; a new source geometry uploads the
 * resize tables with a blocking copy, as in cd_forward_u8.  Neither is legal while `stream` is being
 * captured into a HIP graph: warm the entry point up with one call outside the capture for each
 * (device, dtype class, net_h, source geometry) that will be captured; calls after that queue only
 * the three kernels.  GPUs with an index of 64 or more have no static array (CD_EINVAL). */
int cd_forward_u8_static(cd_handle* h, const uint8_t* src, int n, int H0, int W0,
                         int64_t row_stride, int64_t frame_stride, int chan_order,
                         int net_h, int net_w,
                         float* logits, float* maxv, int64_t* argmax, void* stream);

/* Per-row maximum and its index over scores (device f32 [n][n_classes], row-major).
 * Replaces torch.max(scores, dim=1) at frameID/segmentation.py:37 for callers that hold raw
 * logits.  First maximum wins; a NaN wins over any number (the first NaN), as in torch. */
int cd_max_argmax(cd_handle* h, const float* scores, int64_t n, int n_classes,
                  float* maxv, int64_t* argmax, void* stream);

/* Validation bookkeeping for one batch of labelled frames, accumulated on the device.
 * Replaces the body of the validation loop at training_scripts/supervised_training.py:186-201:
 * pc = torch.max(pred, 1)[1]; correct[c] += #(label == c and pc == c); total[c] += #(label == c);
 * plus the summed cross-entropy of pred against the labels (nn.CrossEntropyLoss, summed over
 * frames rather than averaged per batch).  logits: device f32 [n][n_classes] (n_classes <= 8);
 * labels: device i64 [n], a label outside 0..n_classes-1 is skipped.  correct, total: device
 * i64 [n_classes]; loss_sum: device f64 [1]; all three are added to, not overwritten (the order of
 * the fp64 additions across wavefronts is not fixed). */
int cd_eval_accumulate(cd_handle* h, const float* logits, const int64_t* labels, int64_t n,
                       int n_classes, int64_t* correct, int64_t* total, double* loss_sum,
                       void* stream);

/* ---- Rows of class scores: log probabilities and distillation ------------------------------------------------
 * The four calls below work on rows of scores in device memory, `n_classes` (1 .. 2^30) consecutive elements of
 * `score_type` each, `row_stride` elements between the starts of two rows (0: every row is the same one), any
 * alignment of the rows.  No counterpart in the reference, whose classifier ends at the scores.  z = x / temperature
 * (2^-16 .. 2^16), p = softmax(z); the sums are held in 32 bits whatever the type.  A score of -inf has probability 0;
 * a row of nothing but -inf has no distribution: log probabilities -inf, entropy 0, gradient 0.  A NaN or +inf makes
 * its row's results NaN (the alternatives stay ordered as cd_max_argmax orders: NaN first).  A class id outside
 * 0..n_classes-1 is skipped, as in cd_eval_accumulate.
 * The calls use nothing of the handle but its device: they may overlap with other calls of the same handle, on any
 * streams.  They allocate nothing and may be captured into a HIP graph; `workspace` (cd_rows_workspace bytes of device
 * memory, 16-byte aligned; NULL where that is 0) holds values of one call only while that call's work runs.  Results do not depend on timing: two calls
 * with the same arguments give the same bits.  The same values at another alignment may not: a row's sums are added in an
 * order that depends on where in a 128-byte line it begins (in cd_distill with `grad`, the gradient's row), and on whether
 * `grad` is given. */
enum { CD_T_F32 = 0, CD_T_BF16 = 1, CD_T_F16 = 2 };      /* element types of scores and their gradients */

/* Bytes of device memory that cd_log_probs (`top` alternatives) or cd_distill (top = 0) needs beside its outputs for n
 * rows; 0 for most sizes: only few, long rows are split between workgroups whose results meet there. */
size_t cd_rows_workspace(int64_t n, int n_classes, int score_type, int top);

/* Of every row the log probability of class ids[row] (logp f32 [n]; 0 where the id is skipped), the entropy
 * -sum p ln p (entropy f32 [n]) and the `top` (0 .. 64, at most n_classes) classes with the highest scores and their
 * log probabilities (top_ids i64, top_logp f32 [n][top]; equal scores in the order of their index).  stats f32 [n][2]:
 * the row's largest score and S = sum exp(z - max z), for the backward call (S is relative to max z log2(e) as rounded to 32
 * bits: max z + ln S is ln sum exp z to 2^-24 |max z|).  ids and logp may be NULL together, entropy
 * may be NULL, top_ids and top_logp may be NULL with top = 0. */
int cd_log_probs(cd_handle* h, const void* scores, int score_type, int64_t n, int n_classes, int64_t row_stride,
                 float temperature, const int64_t* ids, int top, float* stats, float* logp, float* entropy,
                 float* top_logp, int64_t* top_ids, void* workspace, size_t workspace_bytes, void* stream);

/* Gradient of sum over rows of grad_logp * logp + grad_entropy * entropy with respect to the scores, rounded once to
 * their type: grad [n][n_classes], grad_stride elements (>= n_classes) between rows.  stats and entropy: of the forward
 * call.  grad_logp (with ids) or grad_entropy (with entropy) may be NULL.  A row that no gradient reaches (its id skipped or
 * its grad_logp 0, and its grad_entropy 0) has gradient 0 whatever its scores.  grad may be the scores' own memory with the
 * scores' stride; otherwise no row of it may overlap with a row of scores (rows of one may lie between rows of the other), nor
 * any with the other arguments. */
int cd_log_probs_backward(cd_handle* h, const void* scores, int score_type, int64_t n, int n_classes,
                          int64_t row_stride, float temperature, const int64_t* ids, const float* stats,
                          const float* entropy, const float* grad_logp, const float* grad_entropy, void* grad,
                          int64_t grad_stride, void* stream);

/* Divergence of every row from a teacher's distribution over `entries` (1 .. 256) classes:
 *   q = softmax(teacher_scores / temperature) over the row's entries, loss = w T^2 sum_j q_j (ln q_j - ln p[id_j])
 * (T^2 keeps the gradient's size independent of the temperature).  teacher_ids i64 [n][entries]: an id outside
 * 0..n_classes-1 marks an unused entry, whose score does not count; a class may be named more than once.  teacher_scores
 * [n][entries] of teacher_type: scores or log probabilities, as cd_log_probs gives them (q does not depend on a constant
 * added to a row).  weights f32 [n] or NULL (all 1): a row of weight 0 is not read, and its loss and gradient are 0, as
 * are those of a row without used entries.  loss f32 [n]; stats f32 [n][2] as in cd_log_probs (-inf and 0 for a row of weight 0).
 * grad: NULL, or [n][n_classes] of score_type for the gradient of the sum of the losses: w T (p - q), rounded once. May
 * be the scores' own memory as in cd_log_probs_backward. */
int cd_distill(cd_handle* h, const void* scores, int score_type, int64_t n, int n_classes, int64_t row_stride,
               float temperature, const int64_t* teacher_ids, const void* teacher_scores, int teacher_type, int entries,
               const float* weights, float* stats, float* loss, void* grad, int64_t grad_stride, void* workspace,
               size_t workspace_bytes, void* stream);

/* Gradient of sum over rows of grad_loss * loss, from the stats of the forward call: for losses that are combined
 * further before they are differentiated.  Arguments as above. */
int cd_distill_backward(cd_handle* h, const void* scores, int score_type, int64_t n, int n_classes, int64_t row_stride,
                        float temperature, const int64_t* teacher_ids, const void* teacher_scores, int teacher_type,
                        int entries, const float* weights, const float* stats, const float* grad_loss, void* grad,
                        int64_t grad_stride, void* stream);

/* Run-length encodes a per-frame class stream into segments.
 * Replaces frameID/segmentation.py:39-60 (Segmentation.__init__ after the max).
 * cls (i64 [n]) and maxv (f32 [n]) are device arrays.  Outputs are device arrays of capacity
 * `cap` rows: end, type, runlen, start (i64), mean (f32: per-segment mean of maxv, formed as
 * torch.mean forms it on a CPU float32 slice - see the top of this file), sum (f64, may be NULL:
 * per-segment sum of maxv).  frame_offset is added to every start/end.
 * n_seg: device i64[1], receives the number of segments found (even when it exceeds cap, in
 * which case only the first cap rows are written and the caller must treat it as CD_ECAP). */
int cd_rle(cd_handle* h, const int64_t* cls, const float* maxv, int64_t n, int64_t frame_offset,
           int64_t* end, int64_t* type, int64_t* runlen, int64_t* start, float* mean, double* sum,
           int64_t cap, int64_t* n_seg, void* stream);

/* Fills dst (device u8 [n][H0][W0][3]) with the deterministic synthetic clip used by the
 * benchmark and the tests: frame i has class classes[i] (device u8 [n]: 0 noise, 1 striped
 * green, 2 near-black) and global index first_index + i.  No counterpart in the reference. */
int cd_synth_frames(cd_handle* h, uint8_t* dst, int n, int H0, int W0,
                    const uint8_t* classes, uint32_t seed, int64_t first_index, void* stream);

/* Per-stage device timing.  While enabled, the launches of the selected stages are bracketed by
 * pairs of HIP events on the caller's stream.  `on`: 0 = off, 1 = every stage, otherwise a mask
 * with bit (CD_STAGE_x + 1) set for each stage to time (an event pair costs a few microseconds
 * of stream time, so a benchmark times only the kernel it reports on).  cd_timing_read() waits
 * for the recorded events of `stage`, returns how many launches were bracketed and their summed
 * duration, and forgets them.
 * No counterpart in the reference; used by bench.py for the per-kernel roofline figures. */
int cd_timing_enable(cd_handle* h, int on);
/* Bracket only every `every`-th launch of each selected stage (default 1 = every launch): the
 * reported totals then cover that sample.  No counterpart in the reference. */
int cd_timing_interval(cd_handle* h, int every);
int cd_timing_read(cd_handle* h, int stage, int64_t* launches, double* total_ms);

/* Host-side orphan gluing + adjacent merge on a segment table in host memory, in place.
 * Replaces frameID/segmentation.py:91-166 glue_orphans() and :168-183
 * combine_adjacent_segments().  Arrays hold *n_seg rows on entry; on return *n_seg is the new
 * row count.  steps: bit 0 = glue orphans, bit 1 = merge adjacent, bit 2 = keep a lone orphan.
 * Returns CD_EINVAL with message "index out of bounds" where the reference raises IndexError
 * (segmentation.py:110-116: the table collapsed to a single segment that is still an orphan);
 * with bit 2 set that segment is kept instead and the call succeeds. */
int cd_glue_segments(int64_t* end, int64_t* type, int64_t* runlen, int64_t* start, float* mean,
                     int64_t* n_seg, int64_t real_threshold, int64_t blank_threshold, int steps);

#ifdef __cplusplus
}
#endif
#endif /* CUTDET_H */
