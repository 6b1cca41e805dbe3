/* ur5learn.h -- C ABI of libur5sim.so's learning operators: what a grasp POLICY needs next to the simulator (sampling, log-probabilities, clipped policy loss, preference
 * loss), and 8-bit activation checkpoints for the network's backward pass. The reference trains a Q network only (Grasping_Agent_multidiscrete.py:388-446); its
 * POLICY_RESNET (Modules.py:304-305) ends in logits that nothing there trains or samples: these entry points do.
 *
 * Conventions of ur5sim.h: 0 or a negative code, ur5_last_error() has the text. No handles: every pointer is a HIP device pointer on `device`, every call queues its
 * kernels on `stream` (a hipStream_t; NULL is the default stream) and returns; nothing is allocated, no state is kept, and a call may be captured into a graph. The calling
 * thread's current device is left as it was. Two calls may run at once if their outputs and workspaces differ.
 *
 * Rows of logits: `rows` rows of `actions` logits (dtype UR5_F32 / UR5_F16 / UR5_BF16), neighbouring in memory within a row, `stride` elements from row to row. mask (NULL:
 * everything is allowed): one byte per pixel, non-zero = allowed, mask_len bytes per row (a divisor of actions: action j uses byte j % mask_len), mask_stride bytes from
 * row to row (0: one mask for all). Logits (and reference logits) of actions that are not allowed may hold anything. A logit of -inf is an action of probability 0;
 * NaN or +inf in an allowed place make the row's results NaN. A row COUNTS if its action lies in [0, actions), is allowed and has a logit above -inf. Less than 2^24 rows and
 * pairs, and rows of which a call makes less than 2^24 workgroups. */
#ifndef UR5LEARN_H
#define UR5LEARN_H
#include "ur5sim.h"
#ifdef __cplusplus
extern "C" {
#endif

enum { UR5_F32 = 0, UR5_F16 = 1, UR5_BF16 = 2 };

typedef struct ur5_rows {
  const void* logits;
  const void* ref;            /* reference policy's logits, same dtype and row layout but for ref_stride; NULL where a call has no use for them */
  const uint8_t* mask;
  int64_t stride, ref_stride, mask_stride;
  int64_t rows, actions, mask_len;
  int32_t dtype, device;
  void* stream;
  void* work;                 /* workspace of at least ur5_policy_work_bytes(...) bytes, 16-byte aligned; contents before and after a call mean nothing, except between
                                 ur5_policy_clip_loss and the ur5_policy_clip_grad calls of the same rows (and prefer_loss / prefer_grad), which read it */
  int64_t work_bytes;
} ur5_rows;

/* mask_len: 0 without a mask; pairs: of the preference loss, 0 for the clipped loss, -1 for ur5_policy_sample and ur5_policy_logp, which need less, and nothing (NULL) for short rows.
   0 also for sizes that a call refuses. */
int64_t ur5_policy_work_bytes(int64_t rows, int64_t actions, int64_t mask_len, int64_t pairs);

/* action[i] ~ softmax(row i) among the allowed actions and its log-probability. The draw is a pure function of (offset, gids[i]): the noise of action j is the j-th number of
   sharding.scene_uniform (offset: its scalar key, gids: global scene ids), so a scene draws the same action however the scenes are sharded. Nothing allowed: -1 and 0. */
int ur5_policy_sample(const ur5_rows* r, uint64_t offset, const int64_t* gids, int64_t* action, float* logp);
/* logp[i] of action[i] (0 for an action outside [0, actions), -inf for one that is not allowed) and the row's entropy (NULL: not wanted; 0 where nothing is allowed). */
int ur5_policy_logp(const ur5_rows* r, const int64_t* action, float* logp, float* entropy);

typedef struct ur5_clip {
  const int64_t* action; const float* old_logp; const float* advantage;   /* [rows] */
  float clip_low, clip_high;     /* the ratio is held to [1 - clip_low, 1 + clip_high] */
  float kl_coef, entropy_coef;   /* kl_coef needs ref */
  float grad_scale;              /* a factor of the gradient */
  const float* upstream;         /* another one, on the device; NULL: 1 */
} ur5_clip;
/* loss[1] = mean over the rows that count of -min(r A, clip(r) A) + kl_coef KL(row || ref) - entropy_coef H(row), r = exp(logp - old_logp); logp, kl, entropy [rows] (0 in rows
   that do not count). No counting row: 0. KL is +inf where the reference gives probability 0 to an action whose own is above 0 in 32 bits; without a kl_coef it is only reported. */
int ur5_policy_clip_loss(const ur5_rows* r, const ur5_clip* c, float* loss, float* logp, float* kl, float* entropy);
/* grad [rows][actions] (dense, dtype of the logits) of the loss times grad_scale times *upstream, from the workspace that clip_loss left; rows that do not count get 0. */
int ur5_policy_clip_grad(const ur5_rows* r, const ur5_clip* c, void* grad);
/* both at once, in two (few rows) or three launches. */
int ur5_policy_clip_loss_grad(const ur5_rows* r, const ur5_clip* c, float* loss, float* logp, float* kl, float* entropy, void* grad);

typedef struct ur5_prefer {
  const int64_t* action; const float* ref_logp;   /* [rows] */
  const int64_t* offsets;        /* [2 pairs + 1], ascending: episode k holds the rows offsets[k] .. offsets[k + 1] - 1; episode 2 i is preferred to 2 i + 1 */
  int64_t pairs;
  double beta, label_smoothing;
  float grad_scale;
  const float* upstream;
} ur5_prefer;
/* loss[1] = mean over pairs of (1 - eps) softplus(-margin) + eps softplus(margin), margin = beta ((preferred episode's sum of logp - ref_logp) - (the other's)); margin [pairs].
   Rows that do not count, or belong to no episode, add nothing. A ref_logp of -inf makes its pair's margin infinite; loss and gradient are then their limits. */
int ur5_policy_prefer_loss(const ur5_rows* r, const ur5_prefer* p, float* loss, float* margin);
int ur5_policy_prefer_grad(const ur5_rows* r, const ur5_prefer* p, void* grad);
/* both at once, in two (few rows and pairs), three or four (long episodes) launches. */
int ur5_policy_prefer_loss_grad(const ur5_rows* r, const ur5_prefer* p, float* loss, float* margin, void* grad);

/* 8-bit activation checkpoints: planes [planes][size] of dtype become codes int8 [planes][groups][64] and scales float [planes][groups], groups = ceil(size / 64): scale = the group's
   largest magnitude / 127 (rounded to fp32, and at most the largest s with a finite 127 s), code = the integer nearest to value / scale (ties to even), what a code stands for is code * scale (rounded to fp32).
   A group whose largest magnitude is below 1e-30 is 0; one that holds an infinity or a NaN stands for NaN throughout. Codes behind a plane's end are 0. */
int ur5_act8_pack(const void* x, int dtype, int64_t planes, int64_t size, int8_t* codes, float* scales, int device, void* stream);
int ur5_act8_unpack(const int8_t* codes, const float* scales, int64_t planes, int64_t size, void* x, int dtype, int device, void* stream);
/* ReLU that leaves a bit per value for its backward pass: y = x <= 0 ? 0 : x (a NaN stays) of `count` neighbouring values, dx = dy where x passed (not x <= 0), 0 elsewhere whatever dy
   holds. bits: ceil(count / 512) * 64 bytes, 8-byte aligned, to be read by ur5_act8_relu_grad of the same count and dtype only. Inputs and outputs may not overlap. */
int ur5_act8_relu(const void* x, int dtype, int64_t count, void* y, uint64_t* bits, int device, void* stream);
int ur5_act8_relu_grad(const void* dy, int dtype, const uint64_t* bits, int64_t count, void* dx, int device, void* stream);
/* weight gradient of a pointwise (1 x 1) convolution from its checkpointed input: codes / scales of x [n][cin][size], dy [n][cout][size] (dense, dtype) ->
   dw [cout][cin] = sum over images and pixels of dy x, db [cout] = sum of dy (NULL: not wanted), both fp32; an infinity in dy makes its row of dw NaN. work: ur5_act8_wgrad_work_bytes(...) bytes, 16-byte aligned. */
int64_t ur5_act8_wgrad_work_bytes(int64_t n, int64_t cin, int64_t cout, int64_t size);
int ur5_act8_wgrad(const int8_t* codes, const float* scales, const void* dy, int dtype, int64_t n, int64_t cin, int64_t cout, int64_t size, float* dw, float* db,
                   void* work, int64_t work_bytes, int device, void* stream);
#ifdef __cplusplus
}
#endif
#endif
