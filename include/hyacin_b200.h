/*
 * hyacin_b200.h -- entry points that exist only in the B200-native build.
 *
 * None of them has a counterpart in the reference library; applications that stay within hyacin.h never
 * need this header.  They expose the individual kernels of the quantized-Gram path (so that each stage can
 * be checked in isolation) and the status word of the bounded waits inside the tensor-core kernel.
 * Pointers are device pointers unless stated otherwise; work is enqueued on handle->cudaStream.
 */
#ifndef HYACIN_B200_H_
#define HYACIN_B200_H_

#include <hyacin.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Non-zero if a bounded wait inside a kernel (Gram, product of 4-bit weights, distillation loss) expired on the current device since the
 * word was last cleared (the results of that call are then invalid).  Call after synchronising the stream.
 * No counterpart in the reference (its kernels have no waits). */
uint32_t hyacinB200Status(int32_t clear);

/* Self-test of the bounded waits: runs a one-block kernel that waits, for pollLimit polls (1 .. 65536), on a
 * barrier that nothing ever completes, so the wait expires the way it would inside the Gram or Cholesky kernels:
 * the kernel returns, `code` (non-zero) appears in the status word, and the device stays usable.  Returns 0 if
 * both waiting roles of the kernel reported that they gave up, -1 for bad arguments, -2 otherwise.  Blocks the
 * host.  No counterpart in the reference. */
int32_t hyacinB200SelfTestWait(const hyacinHandle_t* handle, uint32_t pollLimit, uint32_t code);

/* Schedule of one hyacinXherkBatch call with `rows` local rows and quantisation bits u: number of CRT
 * moduli, bytes per biased quantised value, rows reconstructed together, rows per kernel launch.
 * Takes over the role of the reference's cost model (src/hyacin_herk.cpp:11-43) for this build.
 * Describes the schedule these stage hooks work with; for complex input hyacinXherkBatch itself prefers a
 * second moduli set with a square root of -1 (two planes per column, one product over all tiles) whenever
 * that set covers the bit budget, which this query does not report. */
void hyacinB200CrtPlan(int32_t u, int32_t Complex, int64_t rows, int32_t* moduli, int32_t* valueBytes,
                       int32_t* groupRows, int32_t* chunkRows);

/* Bits each row segment really needs: segU[b] = u + max_j (vexp[0][j] - vexp[b + 1][j]) over the columns that are not
 * zero in the segment, INT32_MIN for an all-zero segment; vexp is the (batches + 1) x N table of
 * hyacinXquantizeScaleBatch, segU a device array of `batches` words.  Asynchronous on the handle's stream.
 * Stage counterpart in the reference: src/fp_exponent.cu:67-76 (internal::int8::vector_range). */
void hyacinB200VectorRange(const hyacinHandle_t* handle, int32_t batches, int32_t N, int32_t u, const int32_t* vexp, int32_t* segU);

/* Tile geometry of the residue buffers for an N x N Gram: tile height / width, tile rows, and the number of
 * tiles that touch the upper triangle.  A residue buffer holds moduli * numTiles * tileY * tileX bytes. */
void hyacinB200TileInfo(int32_t N, int32_t* tileY, int32_t* tileX, int32_t* tilesY, int32_t* numTiles);

/* Work schedule of the residue Gram kernel (host mirror, no GPU needed): the k-th item of CTA pair `pair` out of `pairs`
 * when `moduli` planes of tilesX column blocks of 256 are multiplied.  An item is `width` (1 or 2) neighbouring 256 x 256
 * tiles of one tile row: (tileRow, tileCol) and, for width 2, (tileRow, tileCol + 1).  full = 0: tiles tileRow <= tileCol of
 * the upper triangle (pairRows is ignored); full = 1: all pairRows x tilesX tiles.  Returns 0 when the pair has fewer than
 * k + 1 items.  Over all pairs every tile of every plane appears exactly once. */
int32_t hyacinB200GramItem(int32_t tilesX, int32_t pairRows, int32_t full, int32_t moduli, int32_t pairs, int32_t pair, int32_t k,
                           int32_t* modulus, int32_t* tileRow, int32_t* tileCol, int32_t* width);

/* Quantise `rows` rows of A (column-major, lda in elements) into int8 residue planes
 * W[modulus][column][part * ldk + row]; ldk is a multiple of 128 and rows [rows, ldk) are zero-filled.
 * Real input: one part.  Complex input: three parts (re, im, -re).
 * Stage counterpart in the reference: src/quantize_crt_real.cu:63-99, src/quantize_crt_complex.cu:72-110. */
void hyacinB200QuantizeCrt(const hyacinHandle_t* handle, hyacinPrecision_t Atype, int32_t rows, int32_t N,
                           const void* A, int32_t lda, const int32_t* vexp, int32_t moduli, int32_t valueBytes,
                           int8_t* W, int64_t ldk);

/* Residue Gram: residues[m][tile][y][x] (+)= sum_k W[m][y][ka0 + k] * W[m][x][kb0 + k] mod modulus m.
 * kRows, ka0, kb0 multiples of 128; kRows <= 130816.
 * Stage counterpart in the reference: src/hyacin_herk.cpp:163-189 with src/crt_diag_real.cu:13-29. */
void hyacinB200GramResidues(const hyacinHandle_t* handle, int32_t N, int32_t moduli, const int8_t* W, int64_t ldw,
                            int64_t planeStride, int32_t ka0, int32_t kb0, int32_t kRows, int32_t accumulate,
                            uint8_t* residues);

/* Residues -> packed 63-bit-limb integers, Cpanel[orderC][N(N+1)/2] (+)= value.
 * Stage counterpart in the reference: src/crt_reconstruct_real.cu:94-99. */
void hyacinB200Reconstruct(const hyacinHandle_t* handle, int32_t N, int32_t moduli, const uint8_t* residues,
                           int32_t beta, int32_t orderC, uint64_t* Cpanel);

/* Limb route, stage by stage.  hyacinB200QuantizeLimbs writes `order` planes of balanced base-256 digits of
 * rint(a 2^vexp), laid out like the residue planes of hyacinB200QuantizeCrt (order = (u + 9) / 8 digits hold
 * |q| <= 2^u).  hyacinB200GramLimbs adds sum_{i,j} 2^(8(i+j)) W_i^T W_j (rows ka0.. of the A operand, kb0.. of the
 * B operand, kRows rows, order * kRows <= 131071) into one panel of the packed integer Gram (beta = 0 overwrites).
 * Stage counterparts in the reference: src/quantize_limbs.cu:60-79; src/hyacin_herk.cpp:148-161 with
 * src/limbs_diag.cu, src/limbs_cross_real.cu and src/limbs_cross_imag.cu. */
void hyacinB200QuantizeLimbs(const hyacinHandle_t* handle, hyacinPrecision_t Atype, int32_t rows, int32_t N, const void* A,
                             int32_t lda, const int32_t* vexp, int32_t order, int8_t* W, int64_t ldk);
void hyacinB200GramLimbs(const hyacinHandle_t* handle, int32_t N, int32_t order, const int8_t* W, int64_t ldw,
                         int64_t planeStride, int32_t ka0, int32_t kb0, int32_t kRows, int32_t beta, int32_t orderC,
                         uint64_t* Cpanel);

/* hyacinXherkBatch for callers that cannot allocate: same arguments, same exact integer Gram in C, but all
 * scratch (int8 residue planes, residue accumulators) lives in a fixed 64 MiB array that is part of the loaded
 * module instead of coming from handle->mempool.  It is meant for hosts that have handed the whole device to
 * their own arena, or that call from a latency-bound loop where an allocator call is not acceptable.
 * Returns 0 on success; -1 for unsupported arguments or a handle that belongs to another device than the current
 * one; -2 (with a message on stderr) when residues(N, moduli) + one 128-row chunk of planes exceed the array --
 * roughly N > 2000 for FP64 at eps 1e-10; -3 if the array's device address or the handle's status word could
 * not be obtained (the handle must come from hyacinCreate on this device).
 * The first call on a device looks the array's address up, which with lazy module loading is also the moment the
 * driver reserves the 64 MiB: make one call -- zero rows is enough, it launches nothing -- before the host takes
 * the rest of the device memory, and outside any stream capture; from then on the array costs 64 MiB of that
 * device until the process exits.  Calls on one device share the array: keep them on one stream or order them
 * with events; calls whose kernels overlap on the GPU race.  Complex input always uses the three-part schedule;
 * handle->GramMatrixAlgorithm is not consulted.
 * This entry point has no counterpart in the reference, whose hyacinXherkBatch always allocates from the pool. */
int32_t hyacinB200HerkBatchStatic(const hyacinHandle_t* handle, int32_t batches, int32_t segM, int32_t lastM, int32_t N,
                                  hyacinPrecision_t Atype, const void* A, int32_t lda, int32_t u, const int32_t* vexp,
                                  int32_t beta, int32_t orderC, uint64_t* C);

/* Wire format of hyacinAllReduce1Drow for a value of orderA 63-bit limbs summed over `ranks` ranks: the value
 * is cut into `slices` words, the first slices-1 holding widthBits unsigned bits each and the last the signed
 * remainder, so that a plain unsigned 64-bit sum over all ranks cannot overflow.  Host only.
 * Takes over the role of the reference's table of limb counts (src/allreduce_1drow.cu:151). */
void hyacinB200SlicePlan(int32_t orderA, int32_t ranks, int32_t* slices, int32_t* widthBits);

/* Format choice and conversion to floating point straight from the slices of a cross-rank sum: C is cut into the
 * slices that `ranks` ranks would exchange, and the Gram matrix is produced from those without re-assembling the
 * limbs in memory (the route the fits take after their all-reduce).  Gives the bits of hyacinXdequantizeInit +
 * hyacinXdequantize.  Stage counterparts in the reference: src/allreduce_1drow.cu:112-131,
 * src/fp_i63tp_dequantize.cu:17-26,121-129. */
void hyacinB200DequantizeViaSlices(const hyacinHandle_t* handle, int32_t N, int32_t orderC, const uint64_t* C, const int32_t* vexp,
                                   hyacinPrecision_t Atype, int32_t ranks, hyacinPrecision_t* Gtype, void* G, int32_t ldg);

/* Number of kernels this library has launched in the calling process (optionally reset to zero).
 * No counterpart in the reference. */
int64_t hyacinB200LaunchCount(int32_t reset);

/* In-situ kernel timing: while enabled, every quantise and Gram launch, the pivoted-Cholesky kernel and the
 * SVD call of hyacinXGevd are bracketed by CUDA events on their own stream; hyacinB200ProfileRead waits for
 * them, returns total milliseconds and launch counts of the quantise and Gram kernels, and clears the record;
 * hyacinB200ProfileReadTail does the same for the Cholesky kernel and the SVD call (what either call finds of the
 * other's kinds is kept for the other).  Enabling or disabling also clears everything.  No counterpart in the
 * reference (its timer, hyacinSync_TimerSegments, groups work by class, not by kernel). */
void hyacinB200ProfileEnable(int32_t enable);
void hyacinB200ProfileRead(double* gramMs, int32_t* gramLaunches, double* quantizeMs, int32_t* quantizeLaunches);
void hyacinB200ProfileReadTail(double* choleskyMs, int32_t* choleskyLaunches, double* svdMs, int32_t* svdCalls);

/* The truncated pivoted Cholesky of hyacinXGevd / hyacinXGinterp on its own: G (N x N, format Gtype, read only)
 * -> rank, the one-based pivot order jpiv[N], and the factor R[k + x * ldr] = R(k, column jpiv[x] - 1) for
 * k <= x, zero below the diagonal, rank rows, in the Gram's own format.  That is the content the reference's
 * src/hyacin_potrfp.cu:214-272 leaves in the upper triangle of the Gram matrix it overwrites, so the two can be
 * compared bit for bit.  Blocks the host. */
int32_t hyacinB200PivotedCholesky(const hyacinHandle_t* handle, double eps, int32_t N, int32_t K, hyacinPrecision_t Gtype,
                                  const void* G, int32_t ldg, int32_t* jpiv, void* R, int32_t ldr);

/* ---- compressed weight matrices: 4-bit form, products, distillation -----------------------------------------
 * A weight matrix W (M x N, column-major: column j holds the M weights of output j) is kept as 4-bit codes with one
 * scale per (column, segment of segM rows) -- the table of hyacinXquantizeScaleBatch with short segments -- plus, where
 * wanted, the truncated SVD of what that loses: W = Wq + U V^T, V from hyacinTsvdFit on the residual R = W - Wq, U = R V.
 * The products below apply Wq + U V^T or its transpose to a few vectors, the distillation loss measures (and
 * differentiates) what the compressed model's logits lose against the original's.  None of these has a counterpart in
 * the reference.
 *
 * Storage.  Wq(r, j) = scales[j * lds + r / segM] * (q(r, j) - zero), zero = zeros[j * lds + r / segM] (0 .. 15), or 8 when
 * zeros is NULL.  Codes: column j starts at codes + j * ldq (bytes, a multiple of 16 and at least 64 * ceil(M / 128); codes
 * 16-byte aligned) and holds blocks of 128 rows as sixteen little-endian 32-bit words; row 32 i + 8 c + 2 p + h of a
 * block (i, c, p < 4, h < 2) is the nibble p + 4 h of word 4 c + i.  Nibbles of rows >= M are written as 0 and ignored.
 * Types: HYACIN_F32, HYACIN_F16 and HYACIN_B200_BF16 (no other entry point takes the latter).
 * segM: a multiple of 32.  lds >= ceil(M / segM).
 *
 * All calls are asynchronous on handle->cudaStream, may be captured into a CUDA graph, and return 0, -1 for arguments
 * they do not take (message on stderr, nothing launched), or -3 when CUDA refused a launch or an allocation.  The handle
 * has to come from hyacinCreate on the device that is current.  Scratch comes from handle->mempool in stream order.  Outputs do not
 * overlap inputs unless stated.  M, N and T of the products are at most 2^31 - 256, and pointers lie on a boundary of their type.
 * Results do not depend on timing: there are no atomic sums. */
#define HYACIN_B200_BF16 ((hyacinPrecision_t)14)      /* within the values that the enumeration's type can hold, 0 .. 15 */

/* 4-bit form of W (type Wtype, leading dimension ldw).  scales has type Stype.  zeros == NULL: symmetric,
 * s = Stype(max|w| / 7), q = clamp(rint(w / s), -7, 7) + 8.  Otherwise lo = min(0, min w), hi = max(0, max w),
 * s = Stype((hi - lo) / 15), zero = clamp(rint(-lo / s), 0, 15), q = clamp(rint(w / s) + zero, 0, 15).  Quotients are rounded as if
 * exact, ties to even.  A scale of zero gives q = zero (8, or 0), one beyond the largest number of Stype is infinite and gives the same.  A
 * segment that holds a NaN or an infinity gets a NaN scale and q = zero.  R (float, ldr >= M) receives W - Wq when it is not NULL. */
int32_t hyacinB200QuantizeW4(const hyacinHandle_t* handle, hyacinPrecision_t Wtype, int32_t M, int32_t N, const void* W, int32_t ldw,
                             int32_t segM, hyacinPrecision_t Stype, uint8_t* codes, int64_t ldq, void* scales, uint8_t* zeros,
                             int32_t lds, float* R, int32_t ldr);

/* opW 'T': Y (N x T) = Wq^T X + V (U^T X), X (M x T).   opW 'N': Y (M x T) = Wq X + U (V^T X), X (N x T), the gradient of
 * the former to its input.  U is M x rank, V is N x rank; rank 0 leaves the correction out.  scales, X, Y, U and V have type
 * Xtype.  Any T >= 0.  rank <= 2^20.  Sums are held in 32 bits and Y is rounded once.  Besides:
 *   - the 16-bit types round the scaled weights s (q - zero) to 16 bits before the product for opW 'N' and, but for some scale tables,
 *     for T > 8 (half: weights beyond 65504 become infinite there); for opW 'T' and few vectors they are exact, and it is (q - zero) x that
 *     must stay below 2^128 before the scale comes in;
 *   - U^T X (V^T X) is held in 32 bits; where the scaled weights are rounded, bfloat16 rounds it to 16 bits, half does not;
 *   - single precision rounds s (q - zero), or s x, to 32 bits; for opW 'T' and few vectors x below 2^-110 in magnitude loses places.
 * An infinite entry of X gives infinities of the weights' signs, NaN where a weight is zero.  An infinite entry of the factor applied last
 * (V for 'T', U for 'N') may give NaN for an infinity. */
int32_t hyacinB200ProductW4(const hyacinHandle_t* handle, char opW, int32_t M, int32_t N, int32_t T, hyacinPrecision_t Xtype,
                            const uint8_t* codes, int64_t ldq, int32_t segM, const void* scales, const uint8_t* zeros, int32_t lds,
                            const void* X, int32_t ldx, int32_t rank, const void* U, int32_t ldu, const void* V, int32_t ldv,
                            void* Y, int32_t ldy);

/* Distillation from a teacher's top logits.  Column t of Z (N x T, type Ztype) holds the logits of token t over N classes;
 * ids (K x T) and teacher (K x T, float), both with leading dimension ldk, the teacher's K largest logits and their
 * classes.  Entries whose id lies outside [0, N) are skipped (pad with -1); a class listed twice counts with both its
 * probabilities.  With u = z / tau, q = softmax(u) and p = softmax(teacher / tau) over the listed entries,
 *     KL_t = sum_i p_i (log p_i - log q_i).
 * teacherLse != NULL (T floats: log-sum-exp of ALL the teacher's logits over tau) makes p the teacher's true probabilities and
 * everything that is not listed one more outcome: KL_t += p_r log(p_r / q_r), p_r = max(0, 1 - sum p_i), q_r = sum of q outside; p_r = 0
 * when every class is listed.
 * loss[t] = weight[t] * KL_t and dZ (N x T, type Ztype, leading dimension lddz; may be Z itself with lddz == ldz) =
 * weight[t] * dKL_t / dz; weight == NULL means 1; a token with weight 0 is not read and gets loss 0 and a zero gradient.
 * loss, dZ and stats may each be NULL; stats (2 floats per token) is what hyacinB200DistillGrad needs to give the same
 * gradient later, with the weights known by then (NaN for a token that had weight 0).  1e-30 <= tau <= 1e30, 0 <= K <= 1024,
 * 1 <= N <= 2^20; finite logits may have any size.  A NaN among a token's logits makes its loss and gradient NaN.  A student
 * probability of zero under a positive teacher probability gives an infinite loss and a finite gradient. */
int32_t hyacinB200DistillLoss(const hyacinHandle_t* handle, hyacinPrecision_t Ztype, int32_t N, int32_t T, const void* Z, int32_t ldz,
                              int32_t K, const int32_t* ids, const float* teacher, int32_t ldk, double tau, const float* teacherLse,
                              const float* weight, float* loss, float* stats, void* dZ, int32_t lddz);
int32_t hyacinB200DistillGrad(const hyacinHandle_t* handle, hyacinPrecision_t Ztype, int32_t N, int32_t T, const void* Z, int32_t ldz,
                              int32_t K, const int32_t* ids, const float* teacher, int32_t ldk, double tau, const float* teacherLse,
                              const float* weight, const float* stats, void* dZ, int32_t lddz);

#ifdef __cplusplus
}
#endif

#endif /* HYACIN_B200_H_ */
