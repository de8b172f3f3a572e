/*
 * fhecore -- MI355X (gfx950) CKKS-RNS evaluation core, C ABI.
 *
 * Replaces, for the encrypted Mamba decode hot loop, the FIDESlib /
 * OpenFHE `fideslib::CryptoContext<DCRTPoly>` calls that the reference's
 * native executors make (native/fideslib_stage0/src/packed_fideslib.cpp,
 * native/fideslib_stage0/src/stage1_mamba2_decode_fideslib.cpp) and the
 * in-tree CUDA helpers beside them.  Python binds it with ctypes
 * (fhe-mamba_amd/fhemamba_amd/_lib.py).
 *
 * Conventions
 *   - Every function returns FHE_OK (0) or an FHE_ERR_* code; no C++
 *     exception crosses the ABI.  fhe_last_error() returns the message of
 *     the calling thread's last failure.
 *   - RNS data is uint64, limb-major: [poly][limb][N].  Limb j of a
 *     ciphertext at level with `nlimb` limbs is reduced mod q_j.  Ciphertext
 *     and plaintext polys are in evaluation (NTT) form unless stated.
 *   - Moduli index the joint list q_0..q_{L-1}, p_0..p_{K-1}.
 *   - Device work is asynchronous on the context's stream; host buffers
 *     passed to *_upload / *_download / fhe_encode* / fhe_decode are only
 *     read or written during the call (encodes copy their input to a
 *     staging buffer; the others synchronise).
 *   - Where an entry point lets its output alias an input, the result may
 *     occupy new device storage: fhe_poly_data gives the current address.
 *   - Handles are owned by the caller and released explicitly.  One
 *     context is used by one host thread at a time.
 */
#ifndef FHECORE_H
#define FHECORE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  FHE_OK = 0,
  FHE_ERR_ARG = 1,   /* invalid argument or shape mismatch */
  FHE_ERR_HIP = 2,   /* HIP runtime failure */
  FHE_ERR_RANGE = 3, /* value does not fit (encode) */
  FHE_ERR_STATE = 4, /* wrong object state (e.g. key for another context) */
  FHE_ERR_INTERNAL = 5
};

typedef struct fhe_context fhe_context;
typedef struct fhe_poly fhe_poly; /* device RNS poly set [npoly][nlimb][N] */
typedef struct fhe_key fhe_key;   /* hybrid switching key */

const char *fhe_last_error(void);
int fhe_abi_version(void);

/* ---- parameters --------------------------------------------------------
 * FLEXIBLEAUTO Q chain (depth+1 primes) and HYBRID P primes for ring 2^log_n.
 * Replaces CCParams<CryptoContextCKKSRNS> + GenCryptoContext prime choice
 * (native/fideslib_stage0/src/packed_fideslib.cpp:1060-1068,
 *  src/fhemamba/ckks_probes.py:180-189). */
int fhe_gen_moduli(uint32_t log_n, uint32_t depth, uint32_t scale_bits,
                   uint32_t first_bits, uint32_t dnum, uint64_t *q_out,
                   uint64_t *p_out, uint32_t p_cap, uint32_t *num_p);

/* ---- context -----------------------------------------------------------
 * Replaces GenCryptoContext + LoadContext (packed_fideslib.cpp:1060-1090,
 * stage1_mamba2_decode_fideslib.cpp:1224-1277): builds twiddle and basis
 * conversion tables on `device`. */
int fhe_context_create(uint32_t log_n, const uint64_t *q, uint32_t num_q,
                       const uint64_t *p, uint32_t num_p, uint32_t dnum,
                       int device, fhe_context **out);
int fhe_context_destroy(fhe_context *ctx);
/* log_n, num_q (L), num_p (K), dnum (non-empty digits), alpha (limbs/digit) */
int fhe_context_info(const fhe_context *ctx, uint32_t *info5);
/* Allocation requests the library has made in this process (device pool
 * requests, fresh or reused, and device or pinned-host table and staging
 * allocations).  No counterpart in the reference: a memory diagnostic, e.g.
 * to show that a stretch of calls allocated nothing. */
int fhe_alloc_count(uint64_t *count);
/* moduli (L+K) and their primitive 2N-th roots psi (L+K). */
int fhe_context_moduli(const fhe_context *ctx, uint64_t *mods, uint64_t *psi);
/* Run the context's work on a caller stream (a hipStream_t, e.g. torch's
 * current stream); NULL restores the context's own stream. */
int fhe_context_set_stream(fhe_context *ctx, void *hip_stream);
/* Replaces the per-op cudaDeviceSynchronize of packed_fideslib.cpp:40-42. */
int fhe_sync(fhe_context *ctx);

/* ---- profiling -----------------------------------------------------------
 * Bracket every kernel the context launches with HIP events on its stream
 * (the reference's phase timers and --profile-evaluation bracket,
 * packed_fideslib.cpp:1216-1220).  fhe_profile_end synchronises and writes a
 * JSON object {"kernel": [launches, total_ms], ...} into buf (cap bytes). */
int fhe_profile_begin(fhe_context *ctx);
int fhe_profile_end(fhe_context *ctx, char *buf, size_t cap);

/* ---- raw batched kernels on caller device memory ------------------------
 * Forward / inverse negacyclic NTT of data [npoly][nlimb][N] in place; limb
 * j uses modulus limb0 + j.  Replaces FIDESlib NTT_/INTT launches
 * (experiments/ntt_warp_tail/probe.cu:58-66, fideslib_plaintext_rns.cu:119-137). */
int fhe_ntt_forward(fhe_context *ctx, uint64_t *data, uint32_t npoly,
                    uint32_t nlimb, uint32_t limb0);
int fhe_ntt_inverse(fhe_context *ctx, uint64_t *data, uint32_t npoly,
                    uint32_t nlimb, uint32_t limb0);
/* acc[2][nq][N] = sum_i x_i (.) w_i for x [n][2][nq][N], w [n][nq][N]: the
 * plaintext-ciphertext inner product of a BSGS diagonal sum
 * (stage1_mamba2_decode_fideslib.cpp:575-600, packed_fideslib.cpp:447-516). */
int fhe_mac(fhe_context *ctx, const uint64_t *x, const uint64_t *w, uint32_t n,
            uint32_t nq, uint64_t *acc);

/* ---- device polys ------------------------------------------------------ */
int fhe_poly_create(fhe_context *ctx, uint32_t npoly, uint32_t nlimb,
                    fhe_poly **out);
int fhe_poly_destroy(fhe_poly *p);
int fhe_poly_shape(const fhe_poly *p, uint32_t *npoly, uint32_t *nlimb);
/* Device pointer of the [npoly][nlimb][N] array (valid until destroy or a
 * shape change). */
int fhe_poly_data(const fhe_poly *p, uint64_t **dev);
int fhe_poly_upload(fhe_poly *p, const uint64_t *host, uint32_t npoly,
                    uint32_t nlimb);
int fhe_poly_download(const fhe_poly *p, uint64_t *host);
/* Ciphertext->Clone() (packed_fideslib.cpp:118). */
int fhe_poly_copy(fhe_poly *dst, const fhe_poly *src);
/* Ciphertext SetLevel / level drop: keep the first nlimb limbs
 * (packed_fideslib.cpp:125-126, stage1_mamba2_decode_fideslib.cpp:621-628). */
int fhe_drop_limbs(fhe_poly *out, const fhe_poly *a, uint32_t nlimb);

/* ---- arithmetic (evaluation form; in-place use with out == a is allowed) -
 * EvalAdd / EvalSub (packed_fideslib.cpp:131-149, :571). */
int fhe_add(fhe_poly *out, const fhe_poly *a, const fhe_poly *b);
int fhe_sub(fhe_poly *out, const fhe_poly *a, const fhe_poly *b);
int fhe_negate(fhe_poly *out, const fhe_poly *a);
/* EvalMult(ct, pt) / EvalAdd(ct, pt) with a one-poly plaintext
 * (packed_fideslib.cpp:177-178, stage1_mamba2_decode_fideslib.cpp:1758-1761). */
int fhe_mul_plain(fhe_poly *out, const fhe_poly *ct, const fhe_poly *pt);
int fhe_add_plain(fhe_poly *out, const fhe_poly *ct, const fhe_poly *pt);
/* Per-limb constants c[j] < q_j: EvalMult(ct, double) once the double is
 * scaled to an integer (packed_fideslib.cpp:118), and EvalAdd(ct, double)
 * (packed_fideslib.cpp:162) which adds c[j] to poly 0 only. */
int fhe_mul_const(fhe_poly *out, const fhe_poly *a, const uint64_t *c);
int fhe_add_const(fhe_poly *out, const fhe_poly *a, const uint64_t *c);
/* out = sum_i m_i * xs[i] over count 2-poly ciphertexts, on their first
 * nlimb limbs (each term holds at least nlimb), with integer weights m_i as
 * two's-complement 128-bit values, weights[2i] the low and weights[2i+1]
 * the high word: the Chebyshev leaf sum, a scaled term per basis element
 * added into the accumulator (packed_fideslib.cpp:577-584), in one pass over
 * the terms.  out is [2][nlimb] and may not alias a term. */
int fhe_linear_wsum(fhe_poly *out, const fhe_poly *const *xs, const uint64_t *weights,
                    uint32_t count, uint32_t nlimb);
/* multIntScalar (native/fideslib_stage0/src/fideslib_refresh_correction.hpp:37). */
int fhe_mul_int(fhe_poly *out, const fhe_poly *a, int64_t c);
/* RescaleInPlace, FLEXIBLEAUTO (packed_fideslib.cpp:236): drop the last limb
 * with division by its prime and centred rounding. */
int fhe_rescale(fhe_poly *out, const fhe_poly *a);
/* fhe_rescale of `count` inputs of one shape at once (as[r] into outs[r]):
 * the rescales of one step of the reference's Chebyshev evaluation (the
 * basis powers of one depth before they are multiplied again,
 * src/fhemamba/ckks_probes.py:108-155) sharing one set of launches.
 * Outputs must be distinct and none may be one of the inputs. */
int fhe_rescale_many(fhe_poly *const *outs, const fhe_poly *const *as, uint32_t count);
/* ModRaise, the first step of EvalBootstrap (packed_fideslib.cpp:235-270,
 * stage1_mamba2_decode_fideslib.cpp:2127): limb 0 (mod q0) of every poly
 * of a, centred, lifted to q_0..q_{nlimb-1}; out is [npoly][nlimb]. */
int fhe_mod_raise(fhe_poly *out, const fhe_poly *a, uint32_t nlimb);
/* Tensor product of two 2-poly ciphertexts -> 3 polys (EvalMult core);
 * a == b gives the 3-product square (EvalSquareInPlace,
 * native/fideslib_stage0/src/fideslib_owned_arithmetic.hpp:10-19). */
int fhe_tensor(fhe_poly *out3, const fhe_poly *a, const fhe_poly *b);

/* ---- keys --------------------------------------------------------------
 * A hybrid switching key as [dnum][2][L+K][N] residues (b then a) in
 * evaluation form; loaded once, kept resident in HBM.  Replaces
 * EvalMultKeyGen / EvalRotateKeyGen + LoadContext key upload
 * (packed_fideslib.cpp:1080-1083). */
int fhe_key_load(fhe_context *ctx, const uint64_t *host, fhe_key **out);
/* The inverse of fhe_key_load: the key's residues [dnum][2][L+K][N] in the
 * same standard evaluation form, into `host` (for serialising the
 * evaluation keys of the client/server handoff: SerializeEvalMultKey /
 * SerializeEvalAutomorphismKey, stage1_mamba2_decode_fideslib.cpp:
 * 1466-1477). */
int fhe_key_download(const fhe_key *k, uint64_t *host);
int fhe_key_destroy(fhe_key *k);

/* ---- key switching ----------------------------------------------------
 * Hybrid key switch of one poly a [1][nq][N] -> out [2][nq][N]. */
int fhe_keyswitch(fhe_poly *out, const fhe_poly *a, const fhe_key *key);
/* Relinearize a 3-poly tensor (EvalMult(ct, ct) relinearisation,
 * packed_fideslib.cpp:147-149). */
int fhe_relinearize(fhe_poly *out, const fhe_poly *ct3, const fhe_key *key);
/* fhe_relinearize of `count` 3-poly tensors of one level at once (ct3s[r]
 * into outs[r]): the independent EvalMult relinearisations of one step of
 * the reference's Chebyshev evaluation (the basis powers of one depth and
 * the giant-step products of one tree height, src/fhemamba/ckks_probes.py:
 * 108-155) as one batched ModUp and one batched ModDown.  Outputs must be
 * distinct and none may be one of the tensors. */
int fhe_relinearize_many(fhe_poly *const *outs, const fhe_poly *const *ct3s, uint32_t count,
                         const fhe_key *key);
/* EvalRotate / EvalConjugate: key switch c1, add c0, apply X -> X^galois
 * (packed_fideslib.cpp:207-221, stage1_mamba2_decode_fideslib.cpp:1779-1801,
 *  :2342). */
int fhe_rotate(fhe_poly *out, const fhe_poly *ct, const fhe_key *key,
               uint32_t galois);
/* fhe_rotate without any device allocation, for callers that cannot
 * allocate (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc).  No counterpart in the reference.  Same result
 * as fhe_rotate, word for word.  `out` must already hold [2][nq][N] (it may
 * be `ct`).  Intermediates live in a fixed 128 MiB device array of the
 * library, one per GPU, kept until the process ends: shapes needing more
 * (roughly N*(dnum_eff*(nq+K) + 3nq + 2K) words, + 2nq*N when out == ct)
 * give FHE_ERR_ARG.  The level's conversion tables must already exist (any
 * allocating key switch at that level builds them), else FHE_ERR_STATE.
 * Calls on one GPU share the array and are ordered on it: a call from
 * another stream (another context, or a caller stream) waits on the GPU for
 * the previous call's work before its own, and host threads take turns
 * enqueuing.  The array keeps the last call's contents. */
int fhe_rotate_noalloc(fhe_poly *out, const fhe_poly *ct, const fhe_key *key,
                       uint32_t galois);
/* EvalFastRotationPrecompute: ModUp'd digits of c1, in a new poly handle of
 * shape [dnum_eff][nq+K][N] (native/fideslib_stage0/src/fideslib_rotation_batch.hpp:17). */
int fhe_rotation_precompute(const fhe_poly *ct, fhe_poly **digits);
/* EvalFastRotation over `count` steps sharing one precompute
 * (fideslib_rotation_batch.hpp:18). */
int fhe_rotate_hoisted(const fhe_poly *ct, const fhe_poly *digits,
                       const fhe_key *const *keys, const uint32_t *galois,
                       uint32_t count, fhe_poly *const *outs);
/* EvalRotate over `count` different ciphertexts of one level at once
 * (cts[r] by keys[r] / galois[r] into outs[r]): the per-stream rotations
 * of the reference's Mamba-2 step (src/stage1_mamba2_decode_fideslib.cpp:
 * 3865-3890, 4047-4052: the same rotate-sum step on every state group) as
 * one batched ModUp and one batched ModDown.  Outputs must be distinct; an
 * output may be one of the inputs. */
int fhe_rotate_many(fhe_poly *const *outs, const fhe_poly *const *cts,
                    const fhe_key *const *keys, const uint32_t *galois,
                    uint32_t count);
/* LinearTransformInPlace(ct, rowSize = count, bStep = bstep, pts)
 * (native/fideslib_stage0/patches/fideslib-v2.1.0-linear-transform-api.patch:21-38,
 *  called at src/stage1_mamba2_decode_fideslib.cpp:3517-3531; unfused form
 *  src/packed_fideslib.cpp:447-516):
 *   out = sum_g rot_giant^g( sum_b pts[g*bstep + b] (.) rot_b(ct) )
 * with pts already pre-rotated by the caller for their giant step.
 * baby_keys[b-1] / baby_galois[b-1] rotate by b strides (b = 1..bstep-1; a
 * key may be null when no diagonal uses that baby), all babies from one
 * ModUp; giant_key rotates by bstep strides and is applied by Horner's rule
 * (required when count > bstep).  pts[k] may be null (zero diagonal); at
 * least one must be present.  Plaintexts are one-poly with at least the
 * ciphertext's limbs.  out may be ct. */
int fhe_linear_transform(fhe_poly *out, const fhe_poly *ct,
                         const fhe_poly *const *pts, uint32_t count,
                         uint32_t bstep, const fhe_key *const *baby_keys,
                         const uint32_t *baby_galois, const fhe_key *giant_key,
                         uint32_t giant_galois);
/* The same sum with the caller's pre-rotation and the giant steps folded
 * in (LinearTransformInPlace with a nonzero offset: the ciphertext rotated
 * by `offset` first, packed_fideslib.cpp:447-516; no separate counterpart):
 * baby_keys[b] / baby_galois[b] for b = 0..min(bstep, count)-1 rotate ct by
 * offset + b strides (baby_keys[0] null: baby 0 is ct itself, no offset),
 * all babies from one ModUp, so the offset costs no key switch of its own.
 * n_giant_keys = 1: giant_keys[0] rotates by bstep strides, applied by
 * Horner's rule; n_giant_keys = G - 1 (G = ceil(count / bstep)):
 * giant_keys[g-1] rotates by g * bstep strides and the G - 1 giant
 * rotations run as one batch of independent key switches. */
int fhe_linear_transform_hoisted(fhe_poly *out, const fhe_poly *ct,
                                 const fhe_poly *const *pts, uint32_t count,
                                 uint32_t bstep, const fhe_key *const *baby_keys,
                                 const uint32_t *baby_galois,
                                 const fhe_key *const *giant_keys,
                                 const uint32_t *giant_galois,
                                 uint32_t n_giant_keys);
/* fhe_linear_transform_hoisted of ncts (1..64) ciphertexts cts[i] of one
 * limb count with the same diagonals and keys, into outs[i]: the
 * bootstrap's CoeffToSlot / SlotToCoeff groups of several ciphertexts
 * refreshed at one point of a circuit (the reference's
 * LinearTransformInPlace per ciphertext, packed_fideslib.cpp:447-516, run
 * in each bootstrap of the decoder's state-group refreshes,
 * stage1_mamba2_decode_fideslib.cpp:3952-3967).  One batched ModUp for every ciphertext's babies, their key
 * switches in shared batches, the giant-step rotations of all of them as
 * one set; the same outputs as ncts single calls.  outs must be distinct;
 * an output may be any of the inputs. */
int fhe_linear_transform_hoisted_many(fhe_poly *const *outs,
                                      const fhe_poly *const *cts, uint32_t ncts,
                                      const fhe_poly *const *pts, uint32_t count,
                                      uint32_t bstep,
                                      const fhe_key *const *baby_keys,
                                      const uint32_t *baby_galois,
                                      const fhe_key *const *giant_keys,
                                      const uint32_t *giant_galois,
                                      uint32_t n_giant_keys);

/* ---- encoding -----------------------------------------------------------
 * MakeCKKSPackedPlaintext (packed_fideslib.cpp:204): special inverse FFT of
 * `count` complex values into `slots` slots, scale, round (ties away from
 * zero), RNS lift to nlimb limbs and NTT, all on the GPU
 * (native/fideslib_stage0/src/gpu_special_fft.cu:12-108,
 *  fideslib_plaintext_rns.cu:11-53).  im may be NULL. */
int fhe_encode(fhe_context *ctx, const double *re, const double *im,
               uint32_t count, uint32_t slots, double scale, uint32_t nlimb,
               fhe_poly *out);
/* nvec encodes in one call: row r of re / im (count values each, im may be
 * NULL) into outs[r], each as fhe_encode would write it.  Replaces the
 * reference decoder's look-ahead batches of MakeCKKSPackedPlaintext calls for
 * uncached BSGS diagonals (stage1_mamba2_decode_fideslib.cpp:165-167,
 * :440-447).  The vectors share the FFT, rounding and NTT launches, up to 16
 * per set.  A row whose values may not fit 62 bits after scaling is encoded
 * by the checked single path; FHE_ERR_RANGE names the first that fails (the
 * outputs of earlier rows are then written).  Outputs must be distinct. */
int fhe_encode_many(fhe_context *ctx, const double *re, const double *im,
                    uint32_t count, uint32_t nvec, uint32_t slots, double scale,
                    uint32_t nlimb, fhe_poly *const *outs);
/* Decode a decrypted one-poly plaintext: iNTT, centred CRT, /scale and the
 * forward special FFT (GetRealPackedValue, packed_fideslib.cpp:1227-1236). */
int fhe_decode(fhe_context *ctx, const fhe_poly *pt, uint32_t slots,
               double scale, double *re, double *im);

/* ---- client-side key material and encryption ---------------------------
 * Every sample below is drawn from a stream named by (seed, sample kind,
 * limb / digit).  A new context uses the ChaCha20 family under a 256-bit
 * master key from OS entropy: secure, and the seed is only a per-call
 * label.  fhe_context_set_sampling replaces the master key
 * (FHE_SAMPLING_CHACHA20 with key32 = 32 bytes, or NULL for fresh OS
 * entropy) or selects the seeded family (FHE_SAMPLING_SEEDED, key32 NULL):
 * there the seed alone fixes every sample, which makes keys reproducible
 * for parity tests and NOT secure (a public key reveals the seed).  Takes
 * effect for later calls.  No counterpart in the reference: OpenFHE draws
 * from its own PRNG (packed_fideslib.cpp:1080-1083). */
enum {
  FHE_SAMPLING_CHACHA20 = 0,
  FHE_SAMPLING_SEEDED = 1
};
int fhe_context_set_sampling(fhe_context *ctx, int mode, const uint8_t *key32);
/* Ternary secret (N int64 coefficients) and the public / switching keys
 * derived from it (KeyGen, EvalMultKeyGen, EvalRotateKeyGen:
 * packed_fideslib.cpp:1080-1083). */
int fhe_keygen_secret(fhe_context *ctx, uint64_t seed, int64_t *s_coef);
/* Sparse-ternary secret with exactly h nonzero coefficients (+-1):
 * KeyGen under SetSecretKeyDist(SPARSE_TERNARY), the Mamba-2 decoder's
 * default (native/fideslib_stage0/src/stage1_mamba2_decode_fideslib.cpp:
 * 1225, stage1_mamba2_config.hpp:211).  1 <= h <= N, else FHE_ERR_ARG. */
int fhe_keygen_secret_sparse(fhe_context *ctx, uint64_t seed, uint32_t h,
                             int64_t *s_coef);
int fhe_keygen_public(fhe_context *ctx, const int64_t *s_coef, uint64_t seed,
                      fhe_poly *pk);
int fhe_keygen_relin(fhe_context *ctx, const int64_t *s_coef, uint64_t seed,
                     fhe_key **out);
int fhe_keygen_galois(fhe_context *ctx, const int64_t *s_coef,
                      uint32_t galois, uint64_t seed, fhe_key **out);
/* Encrypt(publicKey, pt) (packed_fideslib.cpp:205) and Decrypt
 * (packed_fideslib.cpp:1227). */
int fhe_encrypt(fhe_poly *ct, const fhe_poly *pk, const fhe_poly *pt,
                uint64_t seed);
int fhe_decrypt(fhe_poly *pt, const fhe_poly *ct, const int64_t *s_coef);

/* ---- Mamba-2 in the clear ------------------------------------------------
 * The layer's operators on plain device memory: what the client runs on its
 * own prompt, and what fits and checks the polynomials (the reference does both
 * in PyTorch on the host, src/fhemamba/reference.py:182-339).  No context:
 * every call takes a hipStream_t of the current device (NULL: its null stream),
 * enqueues there and returns; nothing is allocated and nothing is waited for,
 * so calls may be captured into a graph.  Workspaces are the caller's, of at
 * least the size the *_workspace call gives, 256-byte aligned, and free again
 * when the call's work is done.  Outputs are contiguous and must not overlap
 * inputs; *_step updates its state in place.  Activations are FHE_F32 or
 * FHE_BF16; gates, states, weights and their gradients are 32-bit floats. */
enum { FHE_F32 = 0, FHE_BF16 = 1 };
enum { FHE_MAX_STATES = 128, FHE_MAX_TAPS = 8, FHE_MAX_TOP = 32 };

/* [sequence][token][head or group] of contiguous runs, strides in elements.
 * Where sequences are packed, stride[0] is not used. */
typedef struct {
  const void *data;
  int64_t stride[3];
} fhe_strided;

/* h_t = exp(log_decay_t) h_{t-1} + (write_t x_t) b_t^T,  y_t = h_t c_t + d x_t
 * for every head, h [head_dim][states]; group g of b and c serves heads
 * g * heads / groups and up.  log_decay <= 0 is meant; -infinity forgets the
 * state.  offsets NULL: `seqs` sequences of `tokens` each.  Else the tokens
 * [offsets[i], offsets[i+1]) are sequence i of `tokens` in all; tokens outside
 * of every sequence give zeros.  tokens < 2^31, states <= FHE_MAX_STATES. */
typedef struct {
  uint32_t dtype, seqs, heads, head_dim, states, groups;
  int64_t tokens;
  const int32_t *offsets; /* device, [seqs + 1], or NULL */
  fhe_strided x, b, c;    /* dtype */
  fhe_strided write, log_decay;
  const float *d;       /* [heads] or NULL */
  const float *initial; /* [seqs][heads][head_dim][states], or NULL: zeros */
} fhe_scan_args;

int fhe_ssm_scan_workspace(const fhe_scan_args *args, int backward,
                           size_t *bytes);
/* y [tokens][heads][head_dim] (for each sequence), final_state as `initial`
 * or NULL. */
int fhe_ssm_scan(const fhe_scan_args *args, void *y, float *final_state,
                 void *workspace, size_t bytes, void *hip_stream);
/* From dy (strided as x) and dfinal (as `initial`, or NULL: zeros).  dx as y;
 * dwrite and dlog_decay [tokens][heads]; db and dc [tokens][groups][states] in
 * dtype; dd [heads] or NULL; dinitial as `initial` or NULL.  Sums have a fixed
 * order: the same inputs give the same bits. */
typedef struct {
  fhe_strided dy;
  const float *dfinal;
  void *dx;
  float *dwrite, *dlog_decay;
  void *db, *dc;
  float *dd, *dinitial;
} fhe_scan_grads;
int fhe_ssm_scan_backward(const fhe_scan_args *args,
                          const fhe_scan_grads *grads, void *workspace,
                          size_t bytes, void *hip_stream);

/* One token of each of `requests` requests.  slots [requests] (device, or NULL:
 * 0, 1, ...) names its row of the state [cache][heads][head_dim][states], which
 * is updated in place; no two requests may name one row.  A slot outside of
 * [0, cache) is padding: y is zero and no state changes.  The token strides are
 * the requests'; stride[0] is not used. */
typedef struct {
  uint32_t dtype, requests, cache, heads, head_dim, states, groups;
  const int32_t *slots;
  fhe_strided x, b, c;
  fhe_strided write, log_decay;
  const float *d;
  float *state;
} fhe_ssm_step_args;
int fhe_ssm_step(const fhe_ssm_step_args *args, void *y, void *hip_stream);

/* y_t = act(bias + sum_k weight_k x_{t - taps + 1 + k}) for every channel, act
 * silu or nothing; weight [channels][taps], 2 <= taps <= FHE_MAX_TAPS.  Before a
 * sequence's first token lie its initial inputs [taps - 1][channels], oldest
 * first (NULL: zeros).  Sequences as in fhe_scan_args; stride[2] is not used. */
typedef struct {
  uint32_t dtype, seqs, channels, taps;
  int64_t tokens;
  const int32_t *offsets;
  fhe_strided x;
  const float *weight, *bias; /* bias may be NULL */
  const void *initial;        /* dtype */
  int silu;
} fhe_conv_args;
/* final_state: each sequence's last taps - 1 inputs, as `initial`, or NULL. */
int fhe_causal_conv(const fhe_conv_args *args, void *y, void *final_state,
                    void *hip_stream);
int fhe_causal_conv_workspace(const fhe_conv_args *args, size_t *bytes);
/* dx as y, dweight as weight, dbias [channels] or NULL, dinitial as `initial`
 * or NULL; dfinal is the gradient of final_state, or NULL: zeros. */
typedef struct {
  fhe_strided dy;
  const void *dfinal;
  void *dx;
  float *dweight, *dbias;
  void *dinitial;
} fhe_conv_grads;
int fhe_causal_conv_backward(const fhe_conv_args *args,
                             const fhe_conv_grads *grads, void *workspace,
                             size_t bytes, void *hip_stream);
/* The single-token form on state [cache][taps - 1][channels], slots as in
 * fhe_ssm_step_args. */
typedef struct {
  uint32_t dtype, requests, cache, channels, taps;
  const int32_t *slots;
  fhe_strided x;
  const float *weight, *bias;
  void *state;
  int silu;
} fhe_conv_step_args;
int fhe_causal_conv_step(const fhe_conv_step_args *args, void *y,
                         void *hip_stream);

/* Rows of logits [rows][vocab] (row_stride elements apart): the log probability
 * of each row's target, the entropy of its distribution, its largest logit and
 * the logarithm of the sum of exponentials relative to that, and the `top` <=
 * FHE_MAX_TOP likeliest tokens with their log probabilities, the lower index
 * first among equals.  A logit of -infinity is a token that is not allowed; a
 * row of nothing else has log probability -infinity and entropy 0.  A NaN makes
 * its row's results NaN.  targets (NULL: none) below 0 are left out (log
 * probability 0); one of vocab or more gives NaN. */
typedef struct {
  uint32_t dtype, top;
  int64_t rows, vocab, row_stride;
  const void *logits;
  const int64_t *targets;
} fhe_logprob_args;
typedef struct {
  float *logprob, *entropy, *peak, *log_sum; /* [rows] */
  float *top_logprob;             /* [rows][top] */
  int32_t *top_index;
} fhe_logprob_out;
int fhe_token_logprobs_workspace(const fhe_logprob_args *args, size_t *bytes);
int fhe_token_logprobs(const fhe_logprob_args *args, const fhe_logprob_out *out,
                       void *workspace, size_t bytes, void *hip_stream);
/* dlogits [rows][vocab] in dtype from the gradients of logprob and entropy
 * [rows] (either may be NULL: zeros) and what the forward call gave. */
int fhe_token_logprobs_backward(const fhe_logprob_args *args,
                                const float *peak, const float *log_sum,
                                const float *entropy, const float *dlogprob,
                                const float *dentropy, void *dlogits,
                                void *hip_stream);

/* Rows [rows][channels], `stride` elements apart. */
typedef struct {
  const void *data;
  int64_t stride;
} fhe_rows;

/* y = v / sqrt(mean(v^2) + eps) * weight with v = x silu(gate), or x where there
 * is no gate (data NULL); the mean is over each of `groups` equal parts of the
 * channels.  x and gate in dtype, y [rows][channels] in out_dtype, which is dtype
 * or FHE_BF16.  A part has at most FHE_MAX_ROW channels.  Squares are summed in 32
 * bits: a row whose squares come to 2^128 or more gives zeros, and squares below
 * 2^-126 lose bits.  A row with a value that is not finite has NaN in it. */
enum { FHE_MAX_ROW = 32768 };
typedef struct {
  uint32_t dtype, out_dtype, groups;
  float eps;
  int64_t rows, channels;
  fhe_rows x, gate;
  const float *weight;
} fhe_norm_args;
int fhe_rms_norm(const fhe_norm_args *args, void *y, void *hip_stream);
int fhe_rms_norm_workspace(const fhe_norm_args *args, size_t *bytes);
/* From dy in out_dtype: dx and dgate [rows][channels] in dtype (dgate with a gate
 * only), dweight [channels].  Sums have a fixed order. */
typedef struct {
  fhe_rows dy;
  void *dx, *dgate;
  float *dweight;
} fhe_norm_grads;
int fhe_rms_norm_backward(const fhe_norm_args *args,
                          const fhe_norm_grads *grads, void *workspace,
                          size_t bytes, void *hip_stream);

/* sum = hidden + scale update (scale [channels], or NULL: 1), y the norm of the
 * unrounded sum as above.  hidden and sum in dtype, update and y in out_dtype. */
typedef struct {
  uint32_t dtype, out_dtype;
  float eps;
  uint32_t reserved;
  int64_t rows, channels;
  fhe_rows hidden, update;
  const float *scale, *weight;
} fhe_add_norm_args;
int fhe_add_norm(const fhe_add_norm_args *args, void *sum, void *y,
                 void *hip_stream);
int fhe_add_norm_workspace(const fhe_add_norm_args *args, size_t *bytes);
/* From dy and the gradient of sum (data NULL: zeros).  sum: the forward call's, or
 * NULL; where it serves (32 bits, no scale) hidden and update are not read.
 * dhidden and dupdate [rows][channels] and dscale [channels] may be NULL; dscale
 * is where there is no scale. */
typedef struct {
  fhe_rows dy, dsum;
  const void *sum;
  void *dhidden, *dupdate;
  float *dscale, *dweight;
} fhe_add_norm_grads;
int fhe_add_norm_backward(const fhe_add_norm_args *args,
                          const fhe_add_norm_grads *grads, void *workspace,
                          size_t bytes, void *hip_stream);

/* scale [rows] = max|x| / 127 and values [rows][channels] = the integer nearest
 * to x / scale (even among equals; both quotients rounded to 32 bits first), within
 * -127 .. 127.  A row of zeros has scale 0; one with a value that is not finite has
 * scale NaN and values 0.  channels <= FHE_MAX_ROW. */
typedef struct {
  uint32_t dtype, reserved;
  int64_t rows, channels;
  fhe_rows x;
} fhe_quantize_args;
int fhe_quantize_rows(const fhe_quantize_args *args, int8_t *values,
                      float *scale, void *hip_stream);

/* y = (q weight^T) row_scale scale + bias, q and row_scale those of x's rows as
 * above: [rows][outputs] in dtype.  weight [outputs][inputs], scale and bias
 * [outputs] (bias may be NULL).  The sums of products are exact.  Rows in whole 64
 * times outputs in whole 16 are fewer than 2^34. */
typedef struct {
  uint32_t dtype, reserved;
  int64_t rows, inputs, outputs;
  fhe_rows x;
  const int8_t *weight;
  const float *scale, *bias;
} fhe_int8_args;
int fhe_int8_linear_workspace(const fhe_int8_args *args, size_t *bytes);
int fhe_int8_linear(const fhe_int8_args *args, void *y, void *workspace,
                    size_t bytes, void *hip_stream);

/* y [tokens][channels] = scale weight[id] in dtype; zeros where an id is below 0,
 * NaN where it is vocab or more. */
typedef struct {
  uint32_t dtype;
  float scale;
  int64_t tokens, vocab, channels;
  fhe_rows weight;
  const int64_t *ids;
} fhe_embed_args;
int fhe_embed(const fhe_embed_args *args, void *y, void *hip_stream);
int fhe_embed_workspace(const fhe_embed_args *args, size_t *bytes);
/* dweight [vocab][channels] in dtype: scale times the sum, in 32 bits and in an order
 * that the ids fix, of each id's rows of dy.  weight is not read. */
int fhe_embed_backward(const fhe_embed_args *args, const fhe_rows *dy,
                       void *dweight, void *workspace, size_t bytes,
                       void *hip_stream);

/* A step of a beam search: of all candidates (beam, token) of a request, which
 * have the beam's score plus the token's log probability, the `width` <=
 * FHE_MAX_TOP largest, in order, the lower beam and then the lower token first
 * among equals (scores are 64-bit numbers, good to about 2^-40, until they are
 * rounded for the result): score, parent and token [requests][width].  logits
 * [requests * beams][vocab], row_stride elements apart; beams <= FHE_MAX_TOP,
 * width <= beams * vocab.  A finished beam (finished may be NULL) has the one
 * candidate `end`, at its own score; its logits are not read, nor those of a beam
 * of score -infinity.  Candidates that are not allowed (a logit of -infinity, a
 * beam of score -infinity) have score -infinity.  A NaN or +infinity among a
 * beam's logits or for its score makes its candidates NaN, which come first. */
typedef struct {
  uint32_t dtype, requests, beams, width;
  int64_t vocab, row_stride, end;
  const void *logits;
  const float *scores;
  const uint8_t *finished;
} fhe_beam_args;
typedef struct {
  float *score;
  int32_t *parent, *token;
} fhe_beam_out;
int fhe_beam_select_workspace(const fhe_beam_args *args, size_t *bytes);
int fhe_beam_select(const fhe_beam_args *args, const fhe_beam_out *out,
                    void *workspace, size_t bytes, void *hip_stream);

/* Rows follow their beams in place: row slots[r][j] of every state takes what row
 * slots[r][parent[r][j]] held before the call.  states [count]: an array on the
 * host; each has `cache` contiguous rows of row_bytes <= 2^30, and no two share
 * memory.  parent [requests][beams] and slots (device; slots NULL: r * beams + j).
 * A parent outside of [0, beams) leaves the row as it is, a slot outside of
 * [0, cache) is padding.  No row may be named twice.  `beams` counts the beams
 * before and after: behind a choice of fewer (its width less than its beams) parent
 * goes on with -1. */
typedef struct {
  void *data;
  int64_t row_bytes;
} fhe_state_rows;
int fhe_reorder_states(const fhe_state_rows *states, uint32_t count,
                       uint32_t requests, uint32_t beams, uint32_t cache,
                       const int32_t *parent, const int32_t *slots,
                       void *hip_stream);

#ifdef __cplusplus
}
#endif
#endif
