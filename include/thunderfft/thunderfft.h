/*
 * thunderfft.h -- C ABI of the MI355X (gfx950) ThunderFFT library
 * (libthunderfft_amd.so).
 *
 * The reference (mcrl/thunderfft) is a header-only CUDA C++ template API with
 * no C ABI.  Each entry point below is the plain-pointer form of one
 * reference interface, cited as path:line in the reference tree; the C++
 * template API of the reference is restated on top of these entry points in
 * <thunderfft/thunderfft.hpp>.  No PyTorch or HIP types appear in the
 * signatures: streams are passed as `void*` (a hipStream_t, NULL = the null
 * stream) and buffers as device pointers.
 *
 * Return codes: THFF_OK on success; THFF_EINVAL where the reference throws
 * std::invalid_argument (always before any HIP call); THFF_EIO where it
 * throws std::runtime_error("[ThunderFFT] ...").  thff_last_error() returns
 * the message of the calling thread's last failure.
 */
#ifndef THUNDERFFT_AMD_THUNDERFFT_H
#define THUNDERFFT_AMD_THUNDERFFT_H

#ifdef __cplusplus
extern "C" {
#endif

#define THFF_OK 0
#define THFF_EINVAL (-22)
#define THFF_EIO (-5)

/* Component type T of the reference templates: float (float2 storage) or
 * half (__half2 storage, low = real, high = imaginary). */
#define THFF_FLOAT 0
#define THFF_HALF 1

/* Library version, major*10000 + minor*100 + patch. */
int thff_version(void);

/* Message of the calling thread's last failed call ("" if none). */
const char* thff_last_error(void);

/* ThunderFFTInitialize<T>(N)
 *   reference: include/thunderfft/thunderfft.cuh:55-56,
 *              include/thunderfft/detail/thunderfft_impl_twiddle.cuh:279-327.
 * Builds (or keeps, if it already holds N) the current device's twiddle table
 * for `precision`: N fp32 complex values W[m] = (cos, sin)(2*pi*m/N), computed
 * in fp64 and rounded once.  One N per (device, precision); another N
 * replaces it.  N outside {64,...,4096} (powers of two) -> THFF_EINVAL before
 * any HIP call.  Serialised per precision; not stream ordered: finish every
 * transform that uses the old table before replacing it. */
int thff_initialize(int precision, int n);

/* ThunderFFTFinalize<T>()
 *   reference: include/thunderfft/thunderfft.cuh:62-63,
 *              include/thunderfft/detail/thunderfft_impl_twiddle.cuh:358-378.
 * Frees the current device's table for `precision`; a second call is a no-op.
 * Other devices' tables are untouched. */
int thff_finalize(int precision);

/* ThunderFFT_global<T,N,forward>(d_input, d_output, batch, stream)
 *   reference: include/thunderfft/thunderfft.cuh:150-154,
 *              include/thunderfft/detail/thunderfft_impl_kernel.cuh:6-41.
 * Batched, unnormalized, out-of-place C2C transforms of `batch` contiguous
 * natural-order signals of n complex values (signal b at offset b*n).
 * forward != 0 uses exp(-2*pi*i*n*k/N), forward == 0 exp(+...).
 * Argument checks in the reference's order, all before any HIP call:
 *   unsupported precision or n -> THFF_EINVAL (a static_assert there);
 *   batch < 0 -> THFF_EINVAL; batch == 0 -> THFF_OK without touching the
 *   pointers; null d_input or d_output, or d_input == d_output -> THFF_EINVAL;
 *   a buffer not aligned to its element (8 bytes for float2, 4 bytes for
 *   half2) -> THFF_EINVAL, since no kernel can read a split element.
 * Any element-aligned buffer is accepted, as in the reference: buffers on a
 * 16-byte boundary (every hipMalloc pointer, and every offset of whole
 * transforms of >= 2 values) take the fastest kernels; others take the fp32
 * kernel, whose 16-byte or single-element accesses need no more than the
 * element's alignment.
 * Requires thff_initialize(precision, n) on the current device (THFF_EIO
 * otherwise).  Synchronises `stream` before returning, like the reference. */
int thff_global(int precision, int n, int forward, const void* d_input, void* d_output,
                int batch, void* stream);

/* Same as thff_global without the final stream synchronisation: the launch is
 * enqueued on `stream` and the call returns.  No counterpart in the
 * reference (whose wrapper always synchronises); for callers that time or
 * pipeline transforms.  Same checks and return codes. */
int thff_global_async(int precision, int n, int forward, const void* d_input, void* d_output,
                      int batch, void* stream);

/* Fused circular convolution (no function counterpart in the reference
 * library; the reference ships it as the sample kernel
 * thunder_convN_block_kernel_realin_realout,
 * sample/conv1d/conv1d_fullfft_l4096_thunder.cu:280-331, which this
 * generalises to complex signals, all seven lengths and per-signal filters):
 *   y[b][k] = sum_m x[b][m] * h[f][(k - m) mod n],  f = per_signal_filter ? b : 0,
 * computed as IFFT(FFT(x[b]) * FFT(h[f])) / n in one kernel (forward FFT,
 * pointwise product, inverse FFT and the 1/n scale; the spectra stay on chip).
 * x and y hold batch*n complex values, h holds batch*n (per-signal) or n
 * (shared) values, all in `precision` storage, natural order.  Same checks and
 * return codes as thff_global (y may alias neither x nor h), except that x, h
 * and y must start on a 16-byte boundary (THFF_EINVAL otherwise: the fused
 * kernels move 16-byte vectors only; every offset of whole signals meets it).
 * Requires thff_initialize(precision, n), synchronises `stream` before
 * returning. */
int thff_conv1d(int precision, int n, const void* d_x, const void* d_h, void* d_y, int batch,
                int per_signal_filter, void* stream);

/* thff_conv1d without the final stream synchronisation. */
int thff_conv1d_async(int precision, int n, const void* d_x, const void* d_h, void* d_y,
                      int batch, int per_signal_filter, void* stream);

/* Spectra of `channels` real filters for thff_conv1d_real: for every channel
 * d, spectrum[d][k] = scale * FFT(h[d])[k], k < n, as fp32 complex (8 bytes per
 * value, natural order).  h holds channels*n real fp32 taps, zero-padded to n,
 * for both precisions; `precision` names the convolution the spectra are for
 * (its twiddle table is used).  Replaces the reference's filter-spectrum
 * preparation filter_fft_once (cuFFT C2C + f32_to_h2 + permute_filter_layout*,
 * sample/conv1d/conv1d_fullfft_l4096_thunder.cu:475-497,154-226); scale = 1
 * gives its spectra, scale = 1/n folds the inverse's normalisation in.
 * Requires thff_initialize(precision, n); THFF_EINVAL for a bad precision or
 * length, channels < 0, null or aliased pointers; channels = 0 is a no-op.
 * Synchronises `stream` before returning. */
int thff_conv1d_real_filter(int precision, int n, const void* d_h, void* d_spectrum,
                            int channels, float scale, void* stream);

/* thff_conv1d_real_filter without the final stream synchronisation. */
int thff_conv1d_real_filter_async(int precision, int n, const void* d_h, void* d_spectrum,
                                  int channels, float scale, void* stream);

/* Fused real-input, real-output convolution with one filter per channel (the
 * reference's thunder_convN_block_kernel_realin_realout,
 * sample/conv1d/conv1d_fullfft_l4096_thunder.cu:280-331, launched by run_case
 * :508-515; the reference instantiates n = 256, 1024, 4096 in half, this
 * takes all seven lengths in float or half):
 *   y[b][d] = Re IFFT(FFT(x[b][d]) * spectrum[d])   (unnormalized inverse),
 * x and y real [batch][channels][n] in `precision` storage, spectrum from
 * thff_conv1d_real_filter(precision, n, ...) for the same channels.  With
 * scale = 1 the output is n * (x (*) h), as the reference writes it; with
 * scale = 1/n it is the circular convolution x (*) h.  x and y must be
 * 16-byte aligned.  Same checks and return codes as thff_conv1d (y may alias
 * neither x nor spectrum; channels <= 0 is THFF_EINVAL when batch > 0).
 * Synchronises `stream` before returning. */
int thff_conv1d_real(int precision, int n, const void* d_x, const void* d_spectrum, void* d_y,
                     int batch, int channels, void* stream);

/* thff_conv1d_real without the final stream synchronisation. */
int thff_conv1d_real_async(int precision, int n, const void* d_x, const void* d_spectrum,
                           void* d_y, int batch, int channels, void* stream);

/* Valid 1-D correlation with a short filter, the result of the reference's
 * conv1d_direct_fft_kernel (sample/conv1d/main.cu:38-128, driven by main
 * :207-336 with the definition of :156-174), which tiles it in 64-point FFT
 * windows; here the sum itself, on the matrix cores (a non-finite input value
 * makes NaN of some neighbouring outputs that do not depend on it, up to two
 * 64-byte chunks of values before those that do and the rest of its own chunk
 * after them; the reference's windows spread it over their 64 points):
 *   y[b][i] = sum_{k < filter_len} x[b][i + k] * taps[k],  i < input_len - filter_len + 1,
 * complex, no conjugation.  x holds batch signals of input_len values and y
 * batch outputs of input_len - filter_len + 1 values, both in `precision`
 * storage; taps are filter_len fp32 complex values (float2) for both
 * precisions.  1 <= filter_len <= 64 and input_len >= filter_len (the
 * sample's checks, main.cu:223-230), THFF_EINVAL otherwise; batch < 0, null,
 * aliased or misaligned pointers are THFF_EINVAL, batch = 0 is a no-op.
 * Requires thff_initialize(precision, 64), as the reference's windows do.
 * Synchronises `stream` before returning. */
int thff_conv1d_valid(int precision, const void* d_x, long long input_len, const void* d_taps,
                      int filter_len, void* d_y, int batch, void* stream);

/* thff_conv1d_valid without the final stream synchronisation. */
int thff_conv1d_valid_async(int precision, const void* d_x, long long input_len,
                            const void* d_taps, int filter_len, void* d_y, int batch,
                            void* stream);

/* Fused 2-D circular convolution of `batch` rows x cols row-major images with
 * one shared rows x cols filter (no function counterpart in the reference
 * library; the reference's 2-D convolution is the sample
 * sample/conv2d/thunder.cu:70-207,556-565, row FFT -> column FFT x H ->
 * column IFFT -> row IFFT over one 1024 x 1024 image, and the unbuilt 64 x 64
 * tile sketch sample/conv2d/thunder_tile64.cu:33-208):
 *   y[b][r][c] = sum_{r',c'} x[b][r'][c'] * h[(r - r') mod rows][(c - c') mod cols],
 * computed as IFFT2(FFT2(x[b]) * FFT2(h)) / (rows*cols).  rows = cols = 64 or
 * 128: one fused kernel (forward 2-D FFT, product, inverse) per image, the
 * image on chip.  rows = cols = 1024 (the reference's sample shape): row FFTs
 * x -> y, and of the filter into an 8.25 MiB workspace (up to 4 per device are
 * kept for the streams that call, until thff_finalize leaves neither precision
 * initialised on the device; a further stream takes
 * over one that is not in use; if there is none, and for captured calls, one is
 * allocated and freed stream-ordered, hipMallocAsync), a column pass (FFT,
 * product, inverse FFT) and inverse row FFTs in place in y.  Other shapes -> THFF_EINVAL; requires thff_initialize(precision, rows).
 * x and y hold batch*rows*cols complex values, h rows*cols.  Same checks,
 * return codes and synchronisation as thff_conv1d. */
int thff_conv2d(int precision, int rows, int cols, const void* d_x, const void* d_h, void* d_y,
                int batch, void* stream);

/* thff_conv2d without the final stream synchronisation. */
int thff_conv2d_async(int precision, int rows, int cols, const void* d_x, const void* d_h,
                      void* d_y, int batch, void* stream);

/* thff_conv2d_async that allocates nothing.  No counterpart in the
 * reference: for callers that cannot allocate device memory (code under HIP
 * graph capture, tight serving loops, harnesses that forbid hipMalloc).
 * Same arguments, checks, results and return codes as thff_conv2d_async
 * (enqueued on `stream`, no synchronisation); the 1024 x 1024 form keeps the
 * filter's row spectra in a device array of the library (8.25 MiB per GPU, held
 * until the process ends) instead of a stream-ordered allocation, so images
 * larger than 1024 x 1024 are THFF_EINVAL.  Every call on one GPU shares
 * that array: calls that overlap on one GPU (other streams, other threads)
 * race and must be serialised by the caller.  Requires
 * thff_initialize(precision, rows) on the current device, as thff_conv2d. */
int thff_conv2d_noalloc(int precision, int rows, int cols, const void* d_x, const void* d_h,
                        void* d_y, int batch, void* stream);

/* Snapshot of the current device's twiddle cache for `precision`: the device
 * pointer (NULL when released) and its length (0 when released).  The
 * reference exposes the same state through its device symbols
 * d_twiddle_{f,h} / d_twiddle_N_{f,h}
 * (include/thunderfft/detail/thunderfft_impl_twiddle.cuh:44-68), read by
 * sample/validation/cache_validation.cu:36-50.  Entries are fp32 complex
 * (8 bytes) for both precisions. */
int thff_twiddle_info(int precision, const void** d_table, int* n);

/* Benchmark/test input generator (no reference counterpart; the reference
 * seeds its inputs on the host or with an LCG kernel,
 * sample/bench/paper_fft.cu:27-43).  Writes `count` complex values to
 * d_out in `precision` storage: component c (real of element e is
 * c = 2*(first_element + e), imaginary c + 1) is
 * 2 * (splitmix64(seed ^ c) >> 40) * 2^-24 - 1, exact in fp32, rounded to
 * nearest-even for half.  Asynchronous on `stream`. */
int thff_fill_uniform(int precision, void* d_out, long long count, unsigned long long seed,
                      long long first_element, void* stream);

/* Benchmark helper (no reference counterpart): copies `bytes` (a multiple
 * of 16) from d_src to d_dst with one 16-byte non-temporal load and store per
 * lane, the fastest streaming copy measured on MI355X.  It gives the device's
 * read-plus-write ceiling beside the transforms (bench.py).  Null,
 * misaligned or overlapping buffers and bad sizes -> THFF_EINVAL before any
 * HIP call; bytes = 0 is a no-op.  Asynchronous on `stream`. */
int thff_copy_nt(void* d_dst, const void* d_src, long long bytes, void* stream);

/* ---- Sequence operators beside the long convolutions (no reference counterpart) ----
 *
 * The gated linear recurrence, the other mixer of a sequence model next to the
 * long convolution, and layer norm over rows that lie side by side: the
 * channels where they come last, as before a projection.  (Where the steps come
 * last, as the convolutions have them, a norm over the channels needs a
 * transposed copy.)  They need no thff_initialize.  precision: THFF_FLOAT, THFF_HALF or THFF_BFLOAT16, the
 * type of the values (here real ones: float, half, bfloat16); states, weights,
 * biases and their gradients are fp32 for all three.  Sums, states and
 * statistics are held in fp32 and every output is rounded once, to nearest
 * even.  The same call gives the same bits each time.  Nothing is kept between
 * calls: scratch memory is the caller's, so calls on any streams and captured
 * calls do not meet.  THFF_EINVAL for bad arguments before any HIP call,
 * THFF_EIO for HIP failures; every synchronous call has an _async twin that
 * returns once the work is enqueued on `stream`. */
#define THFF_BFLOAT16 2

/* Layouts of a scan's values: channels last is [batch][n][channels], one row of
 * `channels` values a step; channels first is [batch][channels][n], the
 * convolutions' layout, one row of n values a channel. */
#define THFF_CHANNELS_LAST 0
#define THFF_CHANNELS_FIRST 1

/* What a scan's calls work on.  Strides are elements between the starts of
 * consecutive rows, at least a row's length, or 0 for rows without a gap: with
 * channels last and x_stride = gate_stride = 2 * channels, x and gate are the
 * halves of one projection's rows.  x_stride and gate_stride hold for the
 * gradients of x and the gate too, y_stride for y and its gradient.  batch, n
 * and channels may be 0, and are at most 2^30, batch * channels at most
 * 2^31 - 256 (THFF_EINVAL too where a call has too many steps for its grid).
 * states: rows of the state pool that slots index (unused without slots). */
typedef struct thff_scan_shape {
    int precision, layout;
    int batch, n, channels, states;
    long long x_stride, gate_stride, y_stride;
} thff_scan_shape;

/* Bytes of d_saved (what the forward pass keeps for the backward pass) and of
 * d_workspace (scratch of one call) for a shape; THFF_EINVAL for a bad shape.
 * 0: the pointer may be null. */
long long thff_gated_scan_saved_bytes(const thff_scan_shape* shape);
long long thff_gated_scan_workspace_bytes(const thff_scan_shape* shape);

/* Gated linear recurrence, for every sequence b and channel c, with
 * f[t] = 1 / (1 + exp(-gate[t])):
 *   h[t] = f[t] * h[t-1] + (1 - f[t]) * x[t],   y[t] = h[t],   t < lengths[b].
 * h before the first step is the state d_state_in, and the state after the last
 * one goes to d_state_out; both are fp32 rows of `channels` values, row b for
 * sequence b, or row slots[b] of a pool of shape->states rows.  A slot outside
 * the pool (-1, say) is an empty place: it starts from zero and stores no state.
 * Two places with the same slot race.  d_state_out may be d_state_in
 * (states kept in place); the two must not overlap otherwise.
 * lengths[b] is taken into [0, n]; y is 0 from there on, and x and the gate are
 * not used there, whatever they hold.  Null d_state_in: zeros; null
 * d_state_out, d_saved: not stored; null d_slots: row b; null d_lengths: n each.
 * An infinity in x, or a NaN in x or the gate, makes later outputs of its
 * sequence and channel infinite or NaN, and no others.  A gate of infinity keeps
 * the state, one of minus infinity puts x in its place (a gate below -87.3
 * keeps 2^-126 of the state).  Steps are joined by products of their gates,
 * which are rounded to multiples of 2^-149: what closed gates leave of a state
 * is off by less than 2^-144 of that state (1.6e-5 for the largest float).
 * x, gate and y start on a boundary of their element, states, slots and lengths
 * on 4 bytes, d_saved and d_workspace on 16.  y may alias neither x nor gate
 * (disjoint rows interleaved in one buffer are fine).  Empty batches and
 * channels are no-ops; n = 0 copies the states. */
int thff_gated_scan(const thff_scan_shape* shape, const void* d_x, const void* d_gate, void* d_y,
                    const void* d_state_in, void* d_state_out, const void* d_slots,
                    const void* d_lengths, void* d_saved, void* d_workspace, void* stream);
int thff_gated_scan_async(const thff_scan_shape* shape, const void* d_x, const void* d_gate,
                          void* d_y, const void* d_state_in, void* d_state_out,
                          const void* d_slots, const void* d_lengths, void* d_saved,
                          void* d_workspace, void* stream);

/* Gradients of thff_gated_scan, from dy and the gradient of the final states
 * (d_dstate_out, null: zeros): lam[t] = dy[t] + f[t+1] * lam[t+1], at the last
 * step lam = dy + dstate_out,
 *   dx[t] = (1 - f[t]) * lam[t],   dgate[t] = lam[t] * (h[t-1] - x[t]) * f[t] * (1 - f[t]),
 * both 0 from lengths[b] on, and d_dstate_in = f[0] * lam[0] (null: not stored),
 * dstate_out where the length is 0.  The dstates are [batch][channels], row b
 * for sequence b.  d_saved is what the forward call of the same shape, x, gate
 * and lengths wrote.  dx and dgate may alias no input.  Alignment as above;
 * n = 0 copies dstate_out. */
int thff_gated_scan_backward(const thff_scan_shape* shape, const void* d_dy, const void* d_x,
                             const void* d_gate, const void* d_saved, const void* d_dstate_out,
                             const void* d_lengths, void* d_dx, void* d_dgate, void* d_dstate_in,
                             void* d_workspace, void* stream);
int thff_gated_scan_backward_async(const thff_scan_shape* shape, const void* d_dy,
                                   const void* d_x, const void* d_gate, const void* d_saved,
                                   const void* d_dstate_out, const void* d_lengths, void* d_dx,
                                   void* d_dgate, void* d_dstate_in, void* d_workspace,
                                   void* stream);

/* Layer norm of `rows` rows of `cols` values, `*_stride` elements between the
 * starts of consecutive rows (at least cols, or 0 for cols):
 *   y = (x - mean) * rstd * weight + bias,   rstd = 1 / sqrt(var + eps),
 * mean and var (divided by cols) of the row.  weight and bias are fp32 [cols]
 * (null: ones, zeros); d_mean and d_rstd, fp32 [rows], keep the statistics for
 * the backward pass (null: not stored).  cols >= 1, eps >= 0; rows = 0 is a
 * no-op.  x and y start on a boundary of their element, the fp32 arrays on 4
 * bytes; y may not alias x. */
int thff_layer_norm(int precision, const void* d_x, long long x_stride, const void* d_weight,
                    const void* d_bias, float eps, void* d_y, long long y_stride, void* d_mean,
                    void* d_rstd, long long rows, int cols, void* stream);
int thff_layer_norm_async(int precision, const void* d_x, long long x_stride,
                          const void* d_weight, const void* d_bias, float eps, void* d_y,
                          long long y_stride, void* d_mean, void* d_rstd, long long rows, int cols,
                          void* stream);

/* Bytes of thff_layer_norm_backward's d_workspace (0, as for all rows of more than
 * 16384 columns: may be null). */
long long thff_layer_norm_workspace_bytes(long long rows, int cols);

/* Gradients of thff_layer_norm from dy, x and the statistics: with
 * xh = (x - mean) * rstd and g = dy * weight,
 *   dx = rstd * (g - mean(g) - xh * mean(g * xh)),
 *   dweight = sum over the rows of dy * xh,   dbias = sum over the rows of dy,
 * fp32 [cols], not accumulated (null: not computed; zeros where rows = 0).
 * dx may alias neither dy nor x.  Alignment as above, d_workspace on 16 bytes. */
int thff_layer_norm_backward(int precision, const void* d_dy, long long dy_stride,
                             const void* d_x, long long x_stride, const void* d_mean,
                             const void* d_rstd, const void* d_weight, void* d_dx,
                             long long dx_stride, void* d_dweight, void* d_dbias,
                             void* d_workspace, long long rows, int cols, void* stream);
int thff_layer_norm_backward_async(int precision, const void* d_dy, long long dy_stride,
                                   const void* d_x, long long x_stride, const void* d_mean,
                                   const void* d_rstd, const void* d_weight, void* d_dx,
                                   long long dx_stride, void* d_dweight, void* d_dbias,
                                   void* d_workspace, long long rows, int cols, void* stream);

/* ---- Operators of a state space block (no reference counterpart) ----
 *
 * The mixer beside the gated recurrence that keeps several states a channel, the short
 * convolution that goes before it, and the norm between blocks.  Types, sums, roundings,
 * alignment, return codes and synchronisation are those of the sequence operators above.
 * Values are [batch][n][channels], one row of `channels` values a step; strides are
 * elements between the starts of consecutive rows, at least a row's length, or 0 for rows
 * without a gap.  Sequence b's states are row b of their array, or row slots[b] of a pool
 * of shape->states rows; a slot outside the pool (-1, say) is an empty place, which
 * starts from zero and stores no state, and two places with the same slot race.
 * state_out may be state_in (states kept in place); the two must not overlap otherwise.
 * Nothing else that a call writes, scratch memory included, may be another of its arrays,
 * but for the norm's sums in their residuals' place.
 * lengths[b] is taken into [0, n]; outputs and gradients are 0 from there on, and no
 * input is used there, whatever it holds. */

/* Short causal convolution.  x_stride holds for the gradient of x too, y_stride for y's.
 * width: 2 to 4 taps.  silu: 1 for the activation, 0 for none.  batch, n, channels at
 * most 2^30, batch * channels at most 2^31 - 256. */
typedef struct thff_conv_shape {
    int precision, silu;
    int batch, n, channels, width, states;
    long long x_stride, y_stride;
} thff_conv_shape;

/* Bytes of thff_short_conv_backward's d_workspace (0: may be null), or THFF_EINVAL. */
long long thff_short_conv_workspace_bytes(const thff_conv_shape* shape);

/* For every sequence and channel, with xe the width - 1 values of the state and then x:
 *   p[t] = bias + sum_{k < width} weight[k] * xe[t + k],   y[t] = p / (1 + exp(-p)) or p,
 * t < lengths[b].  weight is fp32 [channels][width], bias fp32 [channels] (null: zeros).
 * A state is [width - 1][channels] values of the shape's type, the last before the next
 * step: state_out is xe's values from lengths[b] on (null: not stored), state_in the
 * same of the call before (null: zeros).  y may not alias x.  Empty batches and channels
 * are no-ops; n = 0 copies the states. */
int thff_short_conv(const thff_conv_shape* shape, const void* d_x, const void* d_weight,
                    const void* d_bias, void* d_y, const void* d_state_in, void* d_state_out,
                    const void* d_slots, const void* d_lengths, void* stream);
int thff_short_conv_async(const thff_conv_shape* shape, const void* d_x, const void* d_weight,
                          const void* d_bias, void* d_y, const void* d_state_in,
                          void* d_state_out, const void* d_slots, const void* d_lengths,
                          void* stream);

/* Gradients of thff_short_conv from dy and that of the last states (d_dstate_out, null:
 * zeros), with dp = dy * (the activation's slope at p):
 *   dxe[e] = sum_k weight[k] * dp[e - k]  (+ dstate_out from e = lengths[b] on),
 *   dweight[k] = sum over all steps of dp[t] * xe[t + k],   dbias = sum of dp,
 * the first width - 1 of dxe to d_dstate_in (null: not stored), the rest to d_dx.
 * d_dweight and d_dbias, fp32, are not accumulated (null: not computed).  The states and
 * their gradients are row b for sequence b, of the shape's type; d_state_in is the
 * forward call's.  d_dx may alias no input, d_workspace starts on 16 bytes. */
int thff_short_conv_backward(const thff_conv_shape* shape, const void* d_dy, const void* d_x,
                             const void* d_weight, const void* d_bias, const void* d_state_in,
                             const void* d_dstate_out, const void* d_lengths, void* d_dx,
                             void* d_dweight, void* d_dbias, void* d_dstate_in,
                             void* d_workspace, void* stream);
int thff_short_conv_backward_async(const thff_conv_shape* shape, const void* d_dy,
                                   const void* d_x, const void* d_weight, const void* d_bias,
                                   const void* d_state_in, const void* d_dstate_out,
                                   const void* d_lengths, void* d_dx, void* d_dweight,
                                   void* d_dbias, void* d_dstate_in, void* d_workspace,
                                   void* stream);

/* State space scan.  order: states of a channel, 1 to 64.  groups divide the channels:
 * channel c has row c / (channels / groups) of b and c, which are [batch][n][groups][order].
 * Each stride holds for the gradient of its array too, and is at most 2^24.  Sizes at
 * most 2^30, batch * channels at most 2^31 - 256 (THFF_EINVAL too where a call has too
 * many workgroups). */
typedef struct thff_state_shape {
    int precision;
    int batch, n, channels, order, groups, states;
    long long x_stride, delta_stride, gate_stride, b_stride, c_stride, y_stride;
} thff_state_shape;

/* Bytes of d_saved (what the forward pass keeps for the backward pass) and of d_workspace
 * (scratch of one call): what a forward call needs (0: may be null), and enough for a call
 * either way; THFF_EINVAL for a bad shape. */
long long thff_state_scan_saved_bytes(const thff_state_shape* shape);
long long thff_state_scan_forward_bytes(const thff_state_shape* shape);
long long thff_state_scan_workspace_bytes(const thff_state_shape* shape);

/* For every sequence and channel, over its states s < order:
 *   dt = log(1 + exp(delta[t] + delta_bias)),
 *   h[t][s] = exp(dt * a[s]) * h[t-1][s] + dt * x[t] * b[t][s],
 *   y[t] = (sum_s c[t][s] * h[t][s] + skip * x[t]) * gate[t] / (1 + exp(-gate[t])),
 * t < lengths[b].  a is fp32 [channels][order], infinite ones count as fp32's largest of
 * their sign (a dt of 0 keeps the state); skip, delta_bias fp32 [channels] (null:
 * zeros); gate null: y without its last factor.  h before the first step is the state
 * d_state_in (null: zeros), after the last one it goes to d_state_out (null: not
 * stored): fp32 rows of [channels][order].  y may alias no input.  Empty batches and
 * channels are no-ops; n = 0 copies the states.  An infinity or a NaN in an input makes
 * later outputs that depend on it infinite or NaN, and no others.  Long sequences may be
 * worked on in segments, each from a state of zero, whose ends are joined: results are
 * as exact as the recurrence of the sizes |state| and |dt * x * b| allows, not that of
 * the states.  The two differ by much only where a is positive and terms that have grown
 * cancel; where the sizes leave fp32's range there, results may be infinite or NaN
 * though the states would not be.  That holds for the gradients too. */
int thff_state_scan(const thff_state_shape* shape, const void* d_x, const void* d_delta,
                    const void* d_a, const void* d_b, const void* d_c, const void* d_skip,
                    const void* d_gate, const void* d_delta_bias, void* d_y,
                    const void* d_state_in, void* d_state_out, const void* d_slots,
                    const void* d_lengths, void* d_saved, void* d_workspace, void* stream);
int thff_state_scan_async(const thff_state_shape* shape, const void* d_x, const void* d_delta,
                          const void* d_a, const void* d_b, const void* d_c, const void* d_skip,
                          const void* d_gate, const void* d_delta_bias, void* d_y,
                          const void* d_state_in, void* d_state_out, const void* d_slots,
                          const void* d_lengths, void* d_saved, void* d_workspace, void* stream);

/* What thff_state_scan_backward reads, and what it writes: pointers on the device.  saved
 * is what the forward call of the same shape and inputs wrote.  dstate_out (null: zeros)
 * and dstate_in (null: not stored) are fp32 [batch][channels][order], row b for sequence
 * b.  dx, ddelta, db, dc and, with a gate, dgate are of the shape's type; da, dskip and
 * ddelta_bias fp32, not accumulated (dskip, ddelta_bias null: not computed).  No output
 * may alias an input or another output. */
typedef struct thff_state_gradients {
    const void *dy, *x, *delta, *a, *b, *c, *skip, *gate, *delta_bias, *saved, *dstate_out,
        *lengths;
    void *dx, *ddelta, *da, *db, *dc, *dskip, *dgate, *ddelta_bias, *dstate_in;
} thff_state_gradients;

/* Gradients of thff_state_scan from dy and that of the last states: with dinner the
 * gradient of the sum before the gate, lam[t] = dinner[t] * c[t] + exp(dt[t+1] * a) * lam[t+1]
 * (dstate_out behind the last step) and q[t] = lam[t] * exp(dt[t] * a) * h[t-1],
 *   dx = dt * sum_s lam * b + dinner * skip,   da = sum over all steps of q * dt,
 *   ddelta = (x * sum_s lam * b + sum_s q * a) / (1 + exp(-(delta + delta_bias))),
 *   db = sum over a group's channels of lam * dt * x,   dc = the same of dinner * h. */
int thff_state_scan_backward(const thff_state_shape* shape, const thff_state_gradients* arrays,
                             void* d_workspace, void* stream);
int thff_state_scan_backward_async(const thff_state_shape* shape,
                                   const thff_state_gradients* arrays, void* d_workspace,
                                   void* stream);

/* Root-mean-square norm of `rows` rows of `cols` values, after a residual's addition:
 *   s = x + residual, rounded to the type of the values,   y = s * rstd * weight,
 * rstd = 1 / sqrt(mean(s^2) + eps).  residual null: s = x.  weight fp32 [cols] (null:
 * ones).  s goes to d_sum (null: not stored), which may be d_residual (the residuals are
 * kept in place, d_sum_stride equal to theirs) and neither x nor y; rstd to d_rstd,
 * fp32 [rows] (null: not stored).  cols >= 1, eps >= 0; rows = 0 is a no-op. */
int thff_rms_norm(int precision, const void* d_x, long long x_stride, const void* d_residual,
                  long long residual_stride, const void* d_weight, float eps, void* d_y,
                  long long y_stride, void* d_sum, long long sum_stride, void* d_rstd,
                  long long rows, int cols, void* stream);
int thff_rms_norm_async(int precision, const void* d_x, long long x_stride,
                        const void* d_residual, long long residual_stride, const void* d_weight,
                        float eps, void* d_y, long long y_stride, void* d_sum,
                        long long sum_stride, void* d_rstd, long long rows, int cols,
                        void* stream);

/* The same with an output of 8 bits (e4m3: 4 exponent bits, 3 of mantissa, finite, 448 the
 * largest): q = y / scale, rounded to nearest even, with a scale for every `block` columns
 * of a row, the largest |y| of them / 448 (at least 2^-126).  block: 128, or cols for one
 * scale a row.  y is rounded once, to q.  q_stride in bytes; d_scales is fp32
 * [rows][ceil(cols / block)].  A NaN in a row makes its q NaN; an infinite y makes its own q
 * NaN, its block's scale infinite and the block's finite values 0. */
int thff_rms_norm_8bit(int precision, const void* d_x, long long x_stride,
                       const void* d_residual, long long residual_stride, const void* d_weight,
                       float eps, void* d_q, long long q_stride, void* d_scales, int block,
                       void* d_sum, long long sum_stride, long long rows, int cols,
                       void* stream);
int thff_rms_norm_8bit_async(int precision, const void* d_x, long long x_stride,
                             const void* d_residual, long long residual_stride,
                             const void* d_weight, float eps, void* d_q, long long q_stride,
                             void* d_scales, int block, void* d_sum, long long sum_stride,
                             long long rows, int cols, void* stream);

/* Bytes of thff_rms_norm_backward's d_workspace (0: may be null). */
long long thff_rms_norm_workspace_bytes(long long rows, int cols);

/* Gradients of thff_rms_norm from dy, the sums s (x itself without a residual) and their
 * rstd, with xh = s * rstd, g = dy * weight and dsum the gradient that reaches s from
 * elsewhere (null: zeros):
 *   dx = rstd * (g - xh * mean(g * xh)) + dsum,   dweight = sum over the rows of dy * xh,
 * dx for x and the residual alike, dweight fp32 [cols], not accumulated (null: not
 * computed; zeros where rows = 0).  dx may alias no input. */
int thff_rms_norm_backward(int precision, const void* d_dy, long long dy_stride,
                           const void* d_sum, long long sum_stride, const void* d_rstd,
                           const void* d_weight, const void* d_dsum, long long dsum_stride,
                           void* d_dx, long long dx_stride, void* d_dweight, void* d_workspace,
                           long long rows, int cols, void* stream);
int thff_rms_norm_backward_async(int precision, const void* d_dy, long long dy_stride,
                                 const void* d_sum, long long sum_stride, const void* d_rstd,
                                 const void* d_weight, const void* d_dsum,
                                 long long dsum_stride, void* d_dx, long long dx_stride,
                                 void* d_dweight, void* d_workspace, long long rows, int cols,
                                 void* stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* THUNDERFFT_AMD_THUNDERFFT_H */
