// HIP kernels (gfx950) for recurrent on-policy training: the gated memory over time, advantages, the clipped policy loss.
// Types: inputs and outputs float32 or bfloat16, states, sums and statistics in 32 bits or more.  Compiled without packed
// float32 instructions.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>

#include "seq_kernels.h"

namespace asmseq {

typedef __bf16 bf16;
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(bf16 x) { return (float)x; }
template <typename T> __device__ __forceinline__ T from_float(float x) { return (T)x; }    // (nearest, ties to even)

#include "kernels_scan.h"
#include "kernels_policy_loss.h"

#define LAUNCH_CHECK() do { hipError_t _e = hipGetLastError(); if (_e != hipSuccess) return (int)_e; } while (0)

namespace {

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool vec_ok(const void *p, int64_t st, int64_t sb, size_t elem, int V) { return !p || (aligned(p, elem * V) && st % V == 0 && sb % V == 0); }

struct Plan { int V, nsplit, Ts; };

constexpr int NW = 4, LF = 8, LB = 4;

// Channels a lane takes and stretches of the time axis.
Plan scan_plan(int64_t T, int64_t C, bool vec)
{
    Plan p{vec && C >= 65536 ? 4 : 1, 1, 0};
    const int64_t groups = (C + 64 * p.V - 1) / (64 * p.V), tile = NW * LF;
    int64_t want = groups >= 256 ? 1 : 512 / groups;
    want = std::min<int64_t>(want, T / (4 * tile));
    want = std::max<int64_t>(1, std::min<int64_t>(want, 64));
    const int64_t tiles = (T + tile - 1) / tile, per = (tiles + want - 1) / want;
    p.Ts = (int)(std::max<int64_t>(per, 1) * tile);
    p.nsplit = (int)std::max<int64_t>(1, (T + p.Ts - 1) / p.Ts);
    return p;
}

template <template <typename, int, bool> class Op, typename T, int V, bool MSK, int L, class Fill>
int scan_go(const ScanGeom &q, Fill fill, hipStream_t st)
{
    Op<T, V, MSK> op;
    fill(op);
    const unsigned groups = (unsigned)((q.C + 64 * V - 1) / (64 * V));
    if (q.nsplit > 1) {
        hipLaunchKernelGGL((k_scan<Op<T, V, MSK>, V, NW, L, true>), dim3(groups, q.nsplit - 1), dim3(64 * NW), 0, st, op, q, (double *)nullptr);
        LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((k_scan<Op<T, V, MSK>, V, NW, L, false>), dim3(groups, q.nsplit), dim3(64 * NW), 0, st, op, q, (double *)nullptr);
    LAUNCH_CHECK();
    return 0;
}
template <template <typename, int, bool> class Op, int L, class Fill>
int scan_dispatch(int dtype, int V, bool msk, const ScanGeom &q, Fill fill, hipStream_t st)
{
#define GO(T, VV) (msk ? scan_go<Op, T, VV, true, L>(q, fill, st) : scan_go<Op, T, VV, false, L>(q, fill, st))
    if (dtype == 0) return V == 4 ? GO(float, 4) : GO(float, 1);
    return V == 4 ? GO(bf16, 4) : GO(bf16, 1);
#undef GO
}

}  // namespace

int64_t scan_workspace(int, int64_t T, int64_t B, int64_t D)
{
    const int64_t C = B * D;                                            // (the larger of the two plans)
    const int n = std::max(scan_plan(T, C, true).nsplit, scan_plan(T, C, false).nsplit);
    return n > 1 ? (int64_t)n * 2 * C * 4 : 0;
}

static ScanGeom scan_geom(const ScanArgs &a, bool vec, int *V)
{
    const Plan p = scan_plan(a.T, a.B * a.D, vec);
    *V = p.V;
    return {(int)a.T, p.nsplit, p.Ts, a.B * a.D, a.D, reinterpret_cast<float *>(a.ws)};
}

int launch_scan_forward(const ScanArgs &a, hipStream_t st)
{
    if (a.B * a.D == 0) return 0;
    const size_t e = a.dtype ? 2 : 4;
    const bool vec = a.D % 4 == 0 && vec_ok(a.gate.p, a.gate.st, a.gate.sb, e, 4) && vec_ok(a.x.p, a.x.st, a.x.sb, e, 4) &&
                     vec_ok(a.out.p, a.out.st, a.out.sb, e, 4) && aligned(a.h0, 16) && aligned(a.h_last, 16) && aligned(a.ws, 16);
    int V;
    const ScanGeom q = scan_geom(a, vec, &V);
    return scan_dispatch<ForwardOp, LF>(a.dtype, V, a.resets || a.lengths, q, [&](auto &op) {
        op.gate = a.gate; op.x = a.x; op.out = a.out; op.h0 = a.h0; op.h_last = a.h_last;
        op.marks = Marks{a.lengths, a.resets, a.r_st, a.r_sb};
    }, st);
}

int launch_scan_backward(const ScanArgs &a, hipStream_t st)
{
    if (a.B * a.D == 0) return 0;
    const size_t e = a.dtype ? 2 : 4;
    const bool vec = a.D % 4 == 0 && vec_ok(a.gate.p, a.gate.st, a.gate.sb, e, 4) && vec_ok(a.x.p, a.x.st, a.x.sb, e, 4) &&
                     vec_ok(a.h.p, a.h.st, a.h.sb, e, 4) && vec_ok(a.dh.p, a.dh.st, a.dh.sb, e, 4) && vec_ok(a.dgate.p, a.dgate.st, a.dgate.sb, e, 4) &&
                     vec_ok(a.dx.p, a.dx.st, a.dx.sb, e, 4) && aligned(a.h0, 16) && aligned(a.dh_last, 16) && aligned(a.dh0, 16) && aligned(a.ws, 16);
    int V;
    const ScanGeom q = scan_geom(a, vec, &V);
    return scan_dispatch<BackwardOp, LB>(a.dtype, V, a.resets || a.lengths, q, [&](auto &op) {
        op.gate = a.gate; op.x = a.x; op.h = a.h; op.dh = a.dh; op.dgate = a.dgate; op.dx = a.dx;
        op.h0 = a.h0; op.dh_last = a.dh_last; op.dh0 = a.dh0;
        op.marks = Marks{a.lengths, a.resets, a.r_st, a.r_sb};
    }, st);
}

int launch_scan_step(int dtype, int64_t B, int64_t D, const void *gate, int64_t g_sb, const void *x, int64_t x_sb, float *state,
                     const uint8_t *reset, int64_t r_sb, void *out, int64_t o_sb, hipStream_t st)
{
    const int64_t n = B * D;
    if (n == 0) return 0;
    const size_t e = dtype ? 2 : 4;
    const bool vec = D % 4 == 0 && vec_ok(gate, 0, g_sb, e, 4) && vec_ok(x, 0, x_sb, e, 4) && vec_ok(out, 0, o_sb, e, 4) && aligned(state, 16);
    const unsigned grid = (unsigned)((n / (vec ? 4 : 1) + 255) / 256);
#define GO(T, V) hipLaunchKernelGGL((k_scan_step<T, V>), dim3(grid), dim3(256), 0, st, n, D, gate, g_sb, x, x_sb, state, reset, r_sb, out, o_sb)
    if (dtype == 0) { if (vec) GO(float, 4); else GO(float, 1); }
    else { if (vec) GO(bf16, 4); else GO(bf16, 1); }
#undef GO
    LAUNCH_CHECK();
    return 0;
}

// [nsplit][2][C] floats, then three doubles a workgroup
int64_t advantages_workspace(int64_t T, int64_t C)
{
    int64_t most = 0;
    for (int v = 0; v < 2; ++v) {
        const Plan p = scan_plan(T, C, v);
        const int64_t groups = (C + 64 * p.V - 1) / (64 * p.V);
        most = std::max(most, (p.nsplit > 1 ? (int64_t)p.nsplit * 2 * C * 4 + 16 : 0) + groups * p.nsplit * 24);
    }
    return most;
}

template <int V, bool MSK, bool MOM> static int advantages_go(const AdvArgs &a, const Plan &p, hipStream_t st)
{
    AdvantageOp<V, MSK, MOM> op;
    op.rewards = a.rewards; op.values = a.values; op.rew_st = a.rew_st; op.val_st = a.val_st; op.done_st = a.done_st;
    op.dones = a.dones; op.lengths = a.lengths; op.gamma = a.gamma; op.lam = a.lam; op.adv = a.adv; op.ret = a.ret; op.C = a.C;
    const unsigned groups = (unsigned)((a.C + 64 * V - 1) / (64 * V));
    ScanGeom q{(int)a.T, p.nsplit, p.Ts, a.C, a.D, reinterpret_cast<float *>(a.ws)};
    double *mom = reinterpret_cast<double *>(reinterpret_cast<char *>(a.ws) + (p.nsplit > 1 ? ((int64_t)p.nsplit * 2 * a.C * 4 + 15) / 16 * 16 : 0));
    if (p.nsplit > 1) {
        hipLaunchKernelGGL((k_scan<AdvantageOp<V, MSK, MOM>, V, NW, LF, true>), dim3(groups, p.nsplit - 1), dim3(64 * NW), 0, st, op, q,
                           (double *)nullptr);
        LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((k_scan<AdvantageOp<V, MSK, MOM>, V, NW, LF, false>), dim3(groups, p.nsplit), dim3(64 * NW), 0, st, op, q, mom);
    LAUNCH_CHECK();
    if (MOM) {
        hipLaunchKernelGGL(k_moments, dim3(1), dim3(256), 0, st, mom, (int64_t)groups * p.nsplit, a.moments);
        LAUNCH_CHECK();
    }
    return 0;
}

int launch_advantages(const AdvArgs &a, hipStream_t st)
{
    const bool vec = a.C % 4 == 0 && vec_ok(a.rewards, a.rew_st, 0, 4, 4) && vec_ok(a.values, a.val_st, 0, 4, 4) &&
                     vec_ok(a.dones, a.done_st, 0, 1, 4) && aligned(a.adv, 16) && aligned(a.ret, 16) && aligned(a.ws, 16);
    const Plan p = scan_plan(a.T, a.C, vec);
    const bool msk = a.dones || a.lengths, mom = a.moments != nullptr;
#define GO(V, M) (mom ? advantages_go<V, M, true>(a, p, st) : advantages_go<V, M, false>(a, p, st))
    if (p.V == 4) return msk ? GO(4, true) : GO(4, false);
    return msk ? GO(1, true) : GO(1, false);
#undef GO
}

namespace {
constexpr int LOSS_GROUPS = 2048, COUNT_GROUPS = 512;
int lanes_of(int A) { return A <= 4 ? 1 : A <= 8 ? 2 : A <= 16 ? 4 : 8; }
int loss_groups(int64_t rows, int A) { return (int)std::min<int64_t>((rows * lanes_of(A) + 255) / 256, LOSS_GROUPS); }
// One workgroup, one launch: what the loss of a minibatch waits for is launches.
bool loss_single(int64_t rows, int A) { return rows * lanes_of(A) <= (A <= 2 ? 4096 : 2048); }
}

int64_t loss_workspace(int64_t rows, int A)
{
    if (loss_single(rows, A)) return 0;
    return (int64_t)loss_groups(rows, A) * (LOSS_SUMS + A) * 8 + COUNT_GROUPS * 8;
}

template <typename TM, int AM, int GL, bool SHARED, bool PACKED> static int loss_go(LossDev p, hipStream_t st)
{
    if (loss_single(p.rows, p.A)) {
        constexpr int BS = AM <= 2 ? 1024 : 512;                        // (the most threads that leave every value in a register)
        hipLaunchKernelGGL((k_policy_loss<TM, AM, GL, SHARED, PACKED, BS>), dim3(1), dim3(BS), 0, st, p);
        LAUNCH_CHECK();
        return 0;
    }
    const int groups = loss_groups(p.rows, p.A);
    if (p.mask.p) {
        p.n_counts = COUNT_GROUPS;
        hipLaunchKernelGGL(k_mask_count, dim3(COUNT_GROUPS), dim3(256), 0, st, p.rows, p.n, p.mask, const_cast<int64_t *>(p.counts));
        LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((k_policy_loss<TM, AM, GL, SHARED, PACKED, 256>), dim3(groups), dim3(256), 0, st, p);
    LAUNCH_CHECK();
    hipLaunchKernelGGL((k_policy_loss_finish<TM, SHARED>), dim3(1), dim3(512), 0, st, p, groups);
    LAUNCH_CHECK();
    return 0;
}
template <typename TM, int AM, int GL> static int loss_pick(const LossDev &p, bool shared, hipStream_t st)
{
    const size_t row = sizeof(TM) * AM;
    const auto packed_rows = [&](const Rows &t) { return AM == 1 || (t.sa == 1 && t.sb % AM == 0 && t.sn % AM == 0 && aligned(t.p, row)); };
    const bool packed = p.A == AM * GL && packed_rows(p.mean) && (shared || packed_rows(p.log_std)) && aligned(p.dmean, row) && (shared || aligned(p.dstd, row));
    if (packed) return shared ? loss_go<TM, AM, GL, true, true>(p, st) : loss_go<TM, AM, GL, false, true>(p, st);
    if constexpr (AM > 1) return shared ? loss_go<TM, AM, GL, true, false>(p, st) : loss_go<TM, AM, GL, false, false>(p, st);
    return -1;
}
template <typename TM> static int loss_width(const LossDev &p, bool shared, hipStream_t st)
{
    if (p.A == 1) return loss_pick<TM, 1, 1>(p, shared, st);
    if (p.A == 2) return loss_pick<TM, 2, 1>(p, shared, st);
    if (p.A <= 4) return loss_pick<TM, 4, 1>(p, shared, st);
    if (p.A <= 8) return loss_pick<TM, 4, 2>(p, shared, st);
    if (p.A <= 16) return loss_pick<TM, 4, 4>(p, shared, st);
    return loss_pick<TM, 4, 8>(p, shared, st);
}

int launch_policy_loss(const LossArgs &a, hipStream_t st)
{
    LossDev p{};
    p.rows = a.B * a.n; p.n = std::max<int64_t>(a.n, 1); p.B = a.B; p.A = a.A;
    p.mean = a.mean; p.log_std = a.log_std; p.actions = a.actions; p.old = a.log_pi_old;
    p.ref = a.log_pi_ref.p ? a.log_pi_ref : a.log_pi_old;
    p.adv = a.adv; p.mask = a.mask; p.moments = a.adv_moments;
    p.lo = 1.0 - a.clip; p.hi = 1.0 + a.clip; p.kl = a.kl_coef; p.ent = a.entropy_coef;
    p.loss = a.loss; p.stats = a.stats; p.dmean = a.dmean; p.dstd = a.dlog_std;
    if (!loss_single(p.rows, p.A)) {
        p.counts = reinterpret_cast<const int64_t *>(a.ws);
        p.part = reinterpret_cast<double *>(a.ws) + COUNT_GROUPS;
    }
    return a.dtype == 0 ? loss_width<float>(p, a.shared_std, st) : loss_width<bf16>(p, a.shared_std, st);
}

int launch_policy_loss_scale(int dtype, const float *grad, int64_t n_mean, void *dmean, int64_t n_std, void *dlog_std, hipStream_t st)
{
    const int64_t n = n_mean + n_std;
    if (n == 0) return 0;
    const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 2048);
    if (dtype == 0) hipLaunchKernelGGL(k_policy_loss_scale<float>, dim3(grid), dim3(256), 0, st, grad, n_mean, (float *)dmean, n_std, (float *)dlog_std);
    else hipLaunchKernelGGL(k_policy_loss_scale<bf16>, dim3(grid), dim3(256), 0, st, grad, n_mean, (bf16 *)dmean, n_std, (bf16 *)dlog_std);
    LAUNCH_CHECK();
    return 0;
}

int launch_gaussian_act(const ActArgs &a, hipStream_t st)
{
    const int64_t rows = a.B * a.n;
    if (rows == 0) return 0;
    const ActDev p{rows, a.n, a.A, 0, a.mean, a.log_std, a.noise, a.actions, a.log_pi};
    const unsigned grid = (unsigned)((rows + 255) / 256);
    if (a.dtype == 0) {
        if (a.noise.p) hipLaunchKernelGGL((k_gaussian_act<float, true>), dim3(grid), dim3(256), 0, st, p);
        else hipLaunchKernelGGL((k_gaussian_act<float, false>), dim3(grid), dim3(256), 0, st, p);
    } else {
        if (a.noise.p) hipLaunchKernelGGL((k_gaussian_act<bf16, true>), dim3(grid), dim3(256), 0, st, p);
        else hipLaunchKernelGGL((k_gaussian_act<bf16, false>), dim3(grid), dim3(256), 0, st, p);
    }
    LAUNCH_CHECK();
    return 0;
}

}  // namespace asmseq
