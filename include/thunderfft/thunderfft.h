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

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* THUNDERFFT_AMD_THUNDERFFT_H */
