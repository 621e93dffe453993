/* b3x_train.h -- the training operators next to the environment step
 * (libb3train.so): what a policy's update needs between the flat arrays that
 * an environment batch writes (observations, rewards, terminals) and the
 * actions that it reads.
 *
 *   b3x_train_logprob_gpu       log probability of each row's action, the row's
 *                               entropy, and its most likely alternatives
 *   b3x_train_logprob_grad_gpu  their gradient with respect to the logits
 *   b3x_train_advantage_gpu     generalised advantages and returns of a rollout
 *   b3x_train_grad_norm_gpu     global norm of a list of gradients, and the
 *                               factor that clips it
 *   b3x_train_adamw_gpu         one AdamW step over a list of tensors, moments
 *                               in 32 bits or in 8
 *
 * Manner of every call: it only enqueues on `stream` and allocates nothing;
 * device memory is the caller's and is used on that stream alone until the
 * enqueued work is done; it returns a cudaError_t code, and where that is
 * cudaErrorInvalidValue nothing was launched or written.  Calls with nothing
 * to do (no rows, no steps, no tensors) succeed without pointers.  Results do
 * not depend on the order in which blocks run: the same inputs give the same
 * bits.
 */
#ifndef B3X_TRAIN_H
#define B3X_TRAIN_H

#include <stddef.h>

#ifdef __cplusplus
#define B3X_TRAIN_API extern "C" __attribute__((visibility("default")))
#else
#define B3X_TRAIN_API __attribute__((visibility("default")))
#endif

/* Element types. */
enum { B3X_F32 = 0, B3X_BF16 = 1, B3X_F16 = 2, B3X_E4M3 = 3, B3X_U8 = 4 };

/* The largest number of alternatives a call returns for a row. */
enum { B3X_TRAIN_MAX_TOP = 32 };

/* Elements that share one scale where moments are held in 8 bits. */
enum { B3X_TRAIN_BLOCK = 256 };

/* For each of `rows` rows z of `width` logits (type B3X_F32, B3X_BF16 or
 * B3X_F16; consecutive in memory, rows `row_stride` elements apart):
 *
 *   m = max z_j,  L = log sum_j exp(scale (z_j - m)),
 *   log p_j = scale (z_j - m) - L,  H = -sum_j p_j log p_j
 *
 *   logp[r]          log p of actions[r] (int32 or int64: action_bytes 4 or 8)
 *   entropy[r]       H
 *   stats[2r]        m, stats[2r + 1] L: what the gradient takes, and with
 *                    scale m + L the log of the row's sum of exponentials
 *   top_ids[r * top + k], top_logp[...]  the `top` largest logits, largest
 *                    first, the lowest index first among equal ones, and
 *                    their log probabilities
 *
 * Outputs that are NULL are not computed.  mask (NULL: none) has `width` bytes
 * a row, rows mask_stride apart (0: one row for all): where its byte is 0 the
 * logit counts as -infinity whatever it holds, NaN included.  A logit of
 * -infinity has probability 0; the lowest finite value is a value like any
 * other.  A row that allows nothing has m = -infinity, L = 0, H = 0, log p =
 * -infinity and no gradient.  An action outside [0, width) stands for "none":
 * its logp is 0.  Alternatives are logits above -infinity; places beyond them
 * hold the index -1 and -infinity.  A NaN or +infinity that is allowed makes
 * the row's m, L, H and log p NaN (m is +infinity for +infinity alone); NaN is
 * never an alternative.  scale (an inverse temperature) is positive and finite.
 * width is at most 2^30; logits and outputs are aligned to their type. */
B3X_TRAIN_API int b3x_train_logprob_gpu(const void* logits, int type, long long rows, long long width,
        long long row_stride, const unsigned char* mask, long long mask_stride, const void* actions,
        int action_bytes, float scale, float* logp, float* entropy, float* stats, int top, int* top_ids,
        float* top_logp, void* stream);

/* The gradient of sum_r (d_logp[r] logp[r] + d_entropy[r] H[r]):
 *
 *   grad_j = scale (d_logp (1[j = action] - p_j) - d_entropy p_j (log p_j + H))
 *
 * from the stats and entropy that b3x_train_logprob_gpu wrote for the same
 * logits, mask and scale.  grad has the logits' type, rows grad_stride apart,
 * and may be the logits themselves (same pointer and stride), not overlap them
 * otherwise.  d_logp or d_entropy (with entropy) may be NULL: zero.  An action
 * that is "none" or has probability 0 by its mask or -infinity takes no
 * d_logp; masked places get 0.  Rounded once, to nearest.  Fastest where a row
 * of grad lies at the same place modulo 16 bytes as its logits. */
B3X_TRAIN_API int b3x_train_logprob_grad_gpu(const void* logits, int type, long long rows, long long width,
        long long row_stride, const unsigned char* mask, long long mask_stride, const void* actions,
        int action_bytes, float scale, const float* stats, const float* entropy, const float* d_logp,
        const float* d_entropy, void* grad, long long grad_stride, void* stream);

/* Generalised advantages of `steps` steps of `envs` environments:
 *
 *   delta_t = r_t + gamma n_t v_{t+1} - v_t,   n_t = 0 where terminal_t != 0, else 1
 *   A_t = delta_t + gamma lam n_t A_{t+1},     R_t = A_t + v_t
 *
 * v after the last step is last_values.  A terminal step takes nothing from
 * beyond it, NaN included, and with a gamma lam of 0 in 32 bits no step takes
 * anything from a later advantage; else a NaN or infinity reaches every step
 * before it.  lengths (NULL: all `steps`) gives each
 * environment's number of steps; last_values follow the last of them, and
 * advantages and returns beyond are 0 whatever the inputs hold there (a length
 * outside [0, steps] counts as the nearer end).  values and last_values have
 * type B3X_F32, B3X_BF16 or B3X_F16, terminals B3X_F32 or B3X_U8; the rest is
 * B3X_F32.  returns may be NULL.  strides, in elements, per step and per
 * environment: rewards, values, terminals (2 each), last_values (1),
 * advantages, returns (2 each).  Outputs overlap nothing.  steps and envs are at
 * most 2^30 each. */
B3X_TRAIN_API int b3x_train_advantage_gpu(long long steps, long long envs, const float* rewards,
        const void* values, int value_type, const void* terminals, int terminal_type, const void* last_values,
        const int* lengths, float* advantages, float* returns, const long long strides[11], float gamma,
        float lam, void* stream);

/* out[0] = the 2-norm of all gradients together, out[1] = min(1, max_norm /
 * (out[0] + 1e-6)), or NaN where the norm is not finite.  Squares are summed
 * in 64 bits, in a fixed order.  workspace: b3x_train_grad_norm_workspace_bytes()
 * bytes, 8-byte aligned, contents of no matter.  max_norm is positive (infinity:
 * no clip). */
B3X_TRAIN_API size_t b3x_train_grad_norm_workspace_bytes(void);
B3X_TRAIN_API int b3x_train_grad_norm_gpu(int count, const void* const* grads, int grad_type,
        const long long* sizes, double max_norm, float* out, void* workspace, size_t workspace_bytes,
        void* stream);

/* One AdamW step of `count` tensors (step counts from 1):
 *
 *   g = grad grad_scale[0];  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
 *   p = p (1 - lr weight_decay) - lr / (1 - beta1^step) m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 *
 * in 32 bits.  For m, v and the square root every operation rounds by itself, so
 * moments, codes and scales are the formula's bits; the parameter is within a few
 * units in the last place of p and of the step taken (fused operations, an
 * approximate reciprocal).  beta1, beta2, eps and the factors made of them and of
 * lr are rounded to 32 bits once.  params: B3X_F32 or B3X_BF16; grads:
 * B3X_F32, B3X_BF16 or B3X_F16; each list of one type, each tensor of sizes[k]
 * consecutive elements, tensors apart from one another.  The pointer arrays,
 * sizes and decays are host memory, read before the call returns.
 *
 * state_type B3X_F32: exp_avg and exp_avg_sq hold m and v.  B3X_E4M3: they hold
 * m and sqrt(v) as e4m3, and scales[k] two floats for each B3X_TRAIN_BLOCK
 * elements, 448 of a code standing for the block's largest: value = code *
 * scale.  A block whose largest is under 2^-100 is held as zeros; sqrt(v) above
 * zero never rounds to zero.  A NaN or infinity makes its whole block's
 * moments NaN (with moments in 32 bits its own alone).
 *
 * copies (NULL: none, or NULL entries): bf16 tensors that get the new
 * parameters, rounded to nearest from 32 bits; parameters that are bf16 and
 * rounded stochastically differ from their copies by up to one spacing of bf16.
 * decays (NULL: weight_decay for all): a weight decay for each tensor.
 * grad_scale (NULL: 1) is read on the device; where it is not finite the whole
 * step leaves everything as it was.
 * stochastic != 0 rounds what is held in fewer than 32 bits (e4m3 moments, bf16
 * parameters) up or down with probabilities in proportion, by a hash of seed,
 * step, the tensor's place in the list and the element; 0 rounds to nearest.
 * Fastest where every array of a tensor starts at a multiple of 4 elements. */
B3X_TRAIN_API int b3x_train_adamw_gpu(int count, void* const* params, int param_type, const void* const* grads,
        int grad_type, void* const* exp_avg, void* const* exp_avg_sq, float* const* scales, int state_type,
        void* const* copies, const long long* sizes, const float* decays, long long step, double lr,
        double beta1, double beta2, double eps, double weight_decay, const float* grad_scale, int stochastic,
        unsigned seed, void* stream);

#endif
