// Internal interface between the C-ABI layer (asm_capi.cpp) and the kernels of recurrent on-policy training
// (seq_kernels.hip).  Not installed; the public interface is include/marl_amd_env.h, group D.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace asmseq {

// One tensor of a sequence operator: element (t, b, d) at p[t * st + b * sb + d].
struct Seq { const void *p; int64_t st, sb; };
struct SeqOut { void *p; int64_t st, sb; };

struct ScanArgs {
    int dtype;                      // ASM_SEQ_F32, ASM_SEQ_BF16
    int64_t T, B, D;
    Seq gate, x, h, dh;             // h: the forward pass's output (backward only)
    const float *h0, *dh_last;
    const uint8_t *resets;          // element (t, b) at resets[t * r_st + b * r_sb]
    int64_t r_st, r_sb;
    const int *lengths;
    SeqOut out, dgate, dx;          // out: h of the forward pass
    float *h_last, *dh0;
    float *kept;                    // the states in front of every eighth step from the end (nullable): written forward, read backward
    void *ws;
};

struct AdvArgs {
    int64_t T, C, D;                // C = channels of one time step (environments x agents), D of them share a length
    const float *rewards, *values;
    int64_t rew_st, val_st, done_st;
    const uint8_t *dones;
    const int *lengths;
    float gamma, lam;
    float *adv, *ret;               // [T][C]
    float *moments;
    void *ws;
};

// One tensor of the policy operators: element (b, i, j) at p[b * sb + i * sn + j * sa].
struct Rows { const void *p; int64_t sb, sn, sa; };

struct LossArgs {
    int dtype, shared_std;
    int64_t B, n;
    int A;
    Rows mean, log_std, actions, log_pi_old, log_pi_ref, adv, mask;
    const float *adv_moments;
    double clip, kl_coef, entropy_coef;
    float *loss, *stats;
    void *dmean, *dlog_std;         // [B][n][A]; [A] or [B][n][A]
    void *ws;
};

struct ActArgs {
    int dtype;
    int64_t B, n;
    int A;
    Rows mean, log_std, noise, actions, log_pi;      // actions: written if noise.p, else read
};

int64_t scan_workspace(int dtype, int64_t T, int64_t B, int64_t D);
int64_t scan_kept(int dtype, int64_t T, int64_t B, int64_t D);
int launch_scan_forward(const ScanArgs &a, hipStream_t st);
int launch_scan_backward(const ScanArgs &a, hipStream_t st);
int launch_scan_step(int dtype, int64_t B, int64_t D, const void *gate, int64_t g_sb, const void *x, int64_t x_sb, float *state,
                     const uint8_t *reset, int64_t r_sb, void *out, int64_t o_sb, hipStream_t st);
int64_t advantages_workspace(int64_t T, int64_t C);
int launch_advantages(const AdvArgs &a, hipStream_t st);
int64_t loss_workspace(int64_t rows, int A);
int launch_policy_loss(const LossArgs &a, hipStream_t st);
int launch_policy_loss_scale(int dtype, const float *grad, int64_t n_mean, void *dmean, int64_t n_std, void *dlog_std, hipStream_t st);
int launch_gaussian_act(const ActArgs &a, hipStream_t st);

}  // namespace asmseq
