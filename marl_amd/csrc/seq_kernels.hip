// HIP kernels (gfx950) for recurrent on-policy training: the gated memory over time, advantages, the clipped policy loss.
// Types: inputs and outputs float32 or bfloat16, states, sums and statistics in 32 bits or more.  Compiled without packed
// float32 instructions.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>

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

// How a scan is laid out: V channels a lane, NW waves that share a tile of time, L steps a wave and tile; nsplit stretches of Ts steps.
struct Plan { int V, NW, L, nsplit, Ts; };

// By C, the channels, and `size`, the bytes of a value (forward + backward of 200 steps, float32 / bfloat16, us):
//   C       1 channel a lane, 4 waves a tile   2 channels, 4 waves   4 channels, one wave walks all of time
//   30720              40 / 35                      42 / 34                     123 / 121
//   62848              77 / 49                      76 / 46                     135 / 122
//   122880            177 / 96                     166 / 85                     165 / 137
//   245760            360 / 196                    357 / 177                    300 / 166
//   491520            704 / 381                    691 / 346                    619 / 324
// Many channels fill the chip by themselves, a wave that shares nothing waits for nobody, and its backward pass needs not read
// h, in float32 either (k_scan_back_kept): from 480 KB a time step on.  Below, four waves side by side in time; from 49152 channels on two of
// them in a lane (half the address work; a backward pass from kept states eight steps a wave and tile).  Rows that are not aligned to
// two or four values go one channel a lane.
// Fewer than 256 workgroups of one channel a lane: what counts is how often a tile's loads are waited for.  Up to `whole` steps eight
// waves share a tile and one launch does it all; from there on the time axis is cut until there are 512 workgroups, down to one tile
// a stretch (1920 channels, forward + backward, us: 100 steps eight waves 14, four 15, cut 15; 200 steps 20, 24, 16; 333 steps
// 27, 34, 19; 2000 steps 111, 166, 42; on the host each of the two launches more costs 4 us or, in a backward pass, up to 20.
// 20011 steps x 183 channels: 61 stretches 97 us, 157 stretches 53 us).
Plan scan_plan(int64_t T, int64_t C, size_t size, bool vec2, bool vec4, int64_t whole = 320)
{
    Plan p{1, 4, 8, 1, 0};
    if (vec4 && C * (int64_t)size >= 480000) p = {4, 1, 4, 1, 0};
    else if (vec2 && C >= 49152) p = {2, 4, 4, 1, 0};
    const int64_t groups = (C + 64 * p.V - 1) / (64 * p.V);
    const bool few = p.V == 1 && groups < 256;
    if (few && T < whole) p.NW = 8;
    const int64_t tile = p.NW * p.L, tiles = std::max<int64_t>(1, (T + tile - 1) / tile);
    int64_t want = 1;
    if (few && T >= whole) want = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(512 / groups, tiles), 256));
    const int64_t per = (tiles + want - 1) / want;
    p.Ts = (int)(per * tile);
    p.nsplit = (int)((tiles + per - 1) / per);
    return p;
}
// (the workspace of any alignment)
int most_splits(int64_t T, int64_t C, size_t size, int64_t whole = 320) { return scan_plan(T, C, size, false, false, whole).nsplit; }

template <int V, int NW, int L, class O> int scan_go(const O &op, const ScanGeom &q, double *mom, hipStream_t st)
{
    const unsigned groups = (unsigned)((q.C + 64 * V - 1) / (64 * V));
    if constexpr (V == 1 && NW == 4)
        if (q.nsplit > 1) {
            const auto agg = op.composing();
            hipLaunchKernelGGL((k_scan<std::remove_const_t<decltype(agg)>, V, NW, L, true>), dim3(groups, q.nsplit - 1), dim3(64 * NW), 0, st, agg, q, (double *)nullptr);
            LAUNCH_CHECK();
        }
    hipLaunchKernelGGL((k_scan<O, V, NW, L, false>), dim3(groups, q.nsplit), dim3(64 * NW), 0, st, op, q, mom);
    LAUNCH_CHECK();
    return 0;
}
template <template <typename, int, bool, typename> class Op, typename T, bool MSK, class Fill>
int scan_typed(const Plan &p, bool far, const ScanGeom &q, Fill fill, hipStream_t st)
{
    constexpr bool BLOCK = Op<T, 1, MSK, uint32_t>::BLOCK;
    if constexpr (!BLOCK)                                               // (with kept states: back_kept())
        if (p.V == 4) { Op<T, 4, MSK, uint32_t> op; fill(op); return scan_go<4, 1, 4>(op, q, nullptr, st); }
    if (p.V == 2) { Op<T, 2, MSK, uint32_t> op; fill(op); return scan_go<2, 4, BLOCK ? 8 : 4>(op, q, nullptr, st); }
    if (far) { Op<T, 1, MSK, int64_t> op; fill(op); return p.NW == 8 ? scan_go<1, 8, 8>(op, q, nullptr, st) : scan_go<1, 4, 8>(op, q, nullptr, st); }
    Op<T, 1, MSK, uint32_t> op;
    fill(op);
    return p.NW == 8 ? scan_go<1, 8, 8>(op, q, nullptr, st) : scan_go<1, 4, 8>(op, q, nullptr, st);
}
template <template <typename, int, bool, typename> class Op, class Fill>
int scan_dispatch(int dtype, bool msk, const Plan &p, bool far, const ScanGeom &q, Fill fill, hipStream_t st)
{
    if (dtype == 0) return msk ? scan_typed<Op, float, true>(p, far, q, fill, st) : scan_typed<Op, float, false>(p, far, q, fill, st);
    return msk ? scan_typed<Op, bf16, true>(p, far, q, fill, st) : scan_typed<Op, bf16, false>(p, far, q, fill, st);
}

// Whether a workgroup's sequences lie too far apart, or backwards, for unsigned 32-bit byte offsets.
bool too_far(int64_t D, std::initializer_list<int64_t> strides, size_t elem)
{
    int64_t sb = 0;
    for (int64_t s : strides) {
        if (s < 0) return true;
        sb = std::max(sb, s);
    }
    const int64_t rows = 64 * 4 / D + 2;
    return (double)rows * (double)sb * (double)elem + (double)D * (double)elem >= 4294967296.0;
}

}  // namespace

int64_t scan_workspace(int dtype, int64_t T, int64_t B, int64_t D)
{
    const int n = most_splits(T, B * D, dtype ? 2 : 4);
    return n > 1 ? (int64_t)n * 2 * B * D * 4 : 0;
}

// Bytes of the states a forward pass keeps for its backward pass, 0 where the pass reads h instead: bfloat16 for the
// gradient's sake, float32 for speed.
int64_t scan_kept(int dtype, int64_t T, int64_t B, int64_t D)
{
    return dtype || (D % 4 == 0 && scan_plan(T, B * D, 4, true, true).NW == 1) ? (T + 7) / 8 * B * D * 4 : 0;
}

static ScanGeom scan_geom(const ScanArgs &a, const Plan &p)
{
    return {(int)a.T, p.nsplit, p.Ts, (uint32_t)(a.B * a.D), (uint32_t)a.D, reinterpret_cast<float *>(a.ws)};
}

int launch_scan_forward(const ScanArgs &a, hipStream_t st)
{
    if (a.B * a.D == 0) return 0;
    const size_t e = a.dtype ? 2 : 4;
    const bool far = too_far(a.D, {a.gate.sb, a.x.sb, a.out.sb, a.r_sb}, e);
    const auto rows = [&](int V) {
        return !far && a.D % V == 0 && vec_ok(a.gate.p, a.gate.st, a.gate.sb, e, V) && vec_ok(a.x.p, a.x.st, a.x.sb, e, V) &&
               vec_ok(a.out.p, a.out.st, a.out.sb, e, V);
    };
    const Plan p = scan_plan(a.T, a.B * a.D, e, rows(2), rows(4));
    return scan_dispatch<ForwardOp>(a.dtype, a.resets || a.lengths, p, far, scan_geom(a, p), [&](auto &op) {
        op.gate = a.gate; op.x = a.x; op.out = a.out; op.h0 = a.h0; op.h_last = a.h_last; op.ck = a.kept;
        op.marks = Marks{a.lengths, a.resets, a.r_st, a.r_sb};
    }, st);
}

template <class Op> static void fill_backward(Op &op, const ScanArgs &a)
{
    op.gate = a.gate; op.x = a.x; op.h = a.h; op.dh = a.dh; op.dgate = a.dgate; op.dx = a.dx;
    op.h0 = a.h0; op.dh_last = a.dh_last; op.dh0 = a.dh0; op.ck = a.kept;
    op.marks = Marks{a.lengths, a.resets, a.r_st, a.r_sb};
}
template <typename T, bool MSK> static int back_kept(const ScanArgs &a, const ScanGeom &q, hipStream_t st)
{
    BackwardKeptOp<T, 4, MSK, uint32_t> op;
    fill_backward(op, a);
    hipLaunchKernelGGL((k_scan_back_kept<T, 4, MSK>), dim3((q.C + 255) / 256), dim3(64), 0, st, op, q);
    LAUNCH_CHECK();
    return 0;
}

int launch_scan_backward(const ScanArgs &a, hipStream_t st)
{
    if (a.B * a.D == 0) return 0;
    const size_t e = a.dtype ? 2 : 4;
    const bool far = too_far(a.D, {a.gate.sb, a.x.sb, a.h.sb, a.dh.sb, a.dgate.sb, a.dx.sb, a.r_sb}, e);
    const auto rows = [&](int V) {
        return !far && a.D % V == 0 && vec_ok(a.gate.p, a.gate.st, a.gate.sb, e, V) && vec_ok(a.x.p, a.x.st, a.x.sb, e, V) && vec_ok(a.h.p, a.h.st, a.h.sb, e, V) &&
               vec_ok(a.dh.p, a.dh.st, a.dh.sb, e, V) && vec_ok(a.dgate.p, a.dgate.st, a.dgate.sb, e, V) && vec_ok(a.dx.p, a.dx.st, a.dx.sb, e, V);
    };
    const Plan p = scan_plan(a.T, a.B * a.D, e, rows(2), rows(4));
    // (the forward pass leaves its states however its own tensors were aligned: these here may be copies of them)
    const bool msk = a.resets || a.lengths;
    if (p.NW == 1 && a.kept && a.T > 0) {
        if (a.dtype == 0) return msk ? back_kept<float, true>(a, scan_geom(a, p), st) : back_kept<float, false>(a, scan_geom(a, p), st);
        return msk ? back_kept<bf16, true>(a, scan_geom(a, p), st) : back_kept<bf16, false>(a, scan_geom(a, p), st);
    }
    const auto fill = [&](auto &op) { fill_backward(op, a); };
    if (a.dtype && a.kept && a.T > 0)
        return msk ? scan_typed<BackwardKeptOp, bf16, true>(p, far, scan_geom(a, p), fill, st) : scan_typed<BackwardKeptOp, bf16, false>(p, far, scan_geom(a, p), fill, st);
    return scan_dispatch<BackwardOp>(a.dtype, msk, p, far, scan_geom(a, p), fill, st);
}

int launch_scan_step(int dtype, int64_t B, int64_t D, const void *gate, int64_t g_sb, const void *x, int64_t x_sb, float *state,
                     const uint8_t *reset, int64_t r_sb, void *out, int64_t o_sb, hipStream_t st)
{
    const int64_t n = B * D;
    if (n == 0) return 0;
    const size_t e = dtype ? 2 : 4;
    const bool vec = D % 4 == 0 && vec_ok(gate, 0, g_sb, e, 4) && vec_ok(x, 0, x_sb, e, 4) && vec_ok(out, 0, o_sb, e, 4) && aligned(state, 16);
    const unsigned grid = (unsigned)((n / (vec ? 4 : 1) + 255) / 256);
#define GO(T, V) hipLaunchKernelGGL((k_scan_step<T, V>), dim3(grid), dim3(256), 0, st, (uint32_t)n, (uint32_t)D, gate, g_sb, x, x_sb, state, reset, r_sb, out, o_sb)
    if (dtype == 0) { if (vec) GO(float, 4); else GO(float, 1); }
    else { if (vec) GO(bf16, 4); else GO(bf16, 1); }
#undef GO
    LAUNCH_CHECK();
    return 0;
}

constexpr int64_t ADV_WHOLE = 160;                                      // (91 channels, whole / cut, us: 96 steps 7.1 / 8.2, 192 steps 8.8 / 8.3, 333 steps 14 / 8.5)

// The stretches' compositions, then three doubles a workgroup.
int64_t advantages_workspace(int64_t T, int64_t C)
{
    const int n = most_splits(T, C, 4, ADV_WHOLE);
    return (n > 1 ? (int64_t)n * 2 * C * 4 + 16 : 0) + (C + 63) / 64 * n * 24;
}

template <int V, int NW, int L, bool MSK, bool MOM> static int advantages_go(const AdvArgs &a, const Plan &p, hipStream_t st)
{
    AdvantageOp<V, MSK, MOM> op;
    op.rewards = a.rewards; op.values = a.values; op.rew_st = a.rew_st; op.val_st = a.val_st; op.done_st = a.done_st;
    op.dones = a.dones; op.lengths = a.lengths; op.gamma = a.gamma; op.lam = a.lam; op.adv = a.adv; op.ret = a.ret; op.C = a.C;
    const unsigned groups = (unsigned)((a.C + 64 * V - 1) / (64 * V));
    ScanGeom q{(int)a.T, p.nsplit, p.Ts, (uint32_t)a.C, (uint32_t)a.D, reinterpret_cast<float *>(a.ws)};
    double *mom = reinterpret_cast<double *>(reinterpret_cast<char *>(a.ws) + (p.nsplit > 1 ? ((int64_t)p.nsplit * 2 * a.C * 4 + 15) / 16 * 16 : 0));
    if (int rc = scan_go<V, NW, L>(op, q, mom, st)) return rc;
    if (MOM) {
        hipLaunchKernelGGL(k_moments, dim3(1), dim3(256), 0, st, mom, (int64_t)groups * p.nsplit, a.moments);
        LAUNCH_CHECK();
    }
    return 0;
}

int launch_advantages(const AdvArgs &a, hipStream_t st)
{
    const auto rows = [&](int V) {
        return a.C % V == 0 && vec_ok(a.rewards, a.rew_st, 0, 4, V) && vec_ok(a.values, a.val_st, 0, 4, V) && vec_ok(a.dones, a.done_st, 0, 1, V) &&
               aligned(a.adv, 4 * V) && aligned(a.ret, 4 * V);
    };
    Plan p = scan_plan(a.T, a.C, 4, false, false, ADV_WHOLE);
    if (rows(4) && a.C >= 49152) p = {4, 4, 4, 1, (int)((a.T + 15) / 16 * 16)};        // (200 x 122880: 75 us; two channels a lane 80 us, one wave for all of time 82 us)
    const bool msk = a.dones || a.lengths, mom = a.moments != nullptr;
#define GO(V, NW, L) (msk ? (mom ? advantages_go<V, NW, L, true, true>(a, p, st) : advantages_go<V, NW, L, true, false>(a, p, st)) \
                          : (mom ? advantages_go<V, NW, L, false, true>(a, p, st) : advantages_go<V, NW, L, false, false>(a, p, st)))
    return p.V == 4 ? GO(4, 4, 4) : p.NW == 8 ? GO(1, 8, 8) : GO(1, 4, 8);
#undef GO
}

namespace {
constexpr int LOSS_GROUPS = 1024, COUNT_GROUPS = 512;
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

template <typename TM, int AM, int GL, bool SHARED, bool LINEAR> static int loss_go(LossDev p, hipStream_t st)
{
    if (loss_single(p.rows, p.A)) {
        constexpr int BS = AM <= 2 && LINEAR ? 1024 : 512;              // (the most threads that leave every value in a register)
        hipLaunchKernelGGL((k_policy_loss<TM, AM, GL, SHARED, LINEAR, BS>), dim3(1), dim3(BS), 0, st, p);
        LAUNCH_CHECK();
        return 0;
    }
    const int groups = loss_groups(p.rows, p.A);
    if (p.mask.p) {
        p.n_counts = COUNT_GROUPS;
        const bool linear = (p.mask.sn == 1 || p.n == 1) && (p.mask.sb == p.n || p.B == 1) && aligned(p.mask.p, 16);
        int64_t *counts = const_cast<int64_t *>(p.counts);
        if (linear) hipLaunchKernelGGL(k_mask_count<true>, dim3(COUNT_GROUPS), dim3(256), 0, st, p.rows, p.n, p.mask, counts);
        else hipLaunchKernelGGL(k_mask_count<false>, dim3(COUNT_GROUPS), dim3(256), 0, st, p.rows, p.n, p.mask, counts);
        LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((k_policy_loss<TM, AM, GL, SHARED, LINEAR, 256>), dim3(groups), dim3(256), 0, st, p);
    LAUNCH_CHECK();
    hipLaunchKernelGGL((k_policy_loss_finish<TM, SHARED>), dim3(1), dim3(512), 0, st, p, groups);
    LAUNCH_CHECK();
    return 0;
}
template <typename TM, int AM, int GL> static int loss_pick(const LossDev &p, bool shared, hipStream_t st)
{
    const size_t row = sizeof(TM) * AM;
    const auto in_line = [&](const Rows &t, int A, size_t align) { return !t.p || ((A == 1 || t.sa == 1) && (t.sn == A || p.n == 1) && (t.sb == (int64_t)p.n * A || p.B == 1) && aligned(t.p, align)); };
    const bool linear = p.A == AM * GL && in_line(p.mean, p.A, row) && (shared || in_line(p.log_std, p.A, row)) && in_line(p.old, 1, 4) && in_line(p.ref, 1, 4) &&
                        in_line(p.adv, 1, 4) && in_line(p.mask, 1, 1) && aligned(p.dmean, row) && (shared || aligned(p.dstd, row));
    if (linear) return shared ? loss_go<TM, AM, GL, true, true>(p, st) : loss_go<TM, AM, GL, false, true>(p, st);
    return shared ? loss_go<TM, AM, GL, true, false>(p, st) : loss_go<TM, AM, GL, false, false>(p, st);
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
    p.rows = (uint32_t)(a.B * a.n); p.n = (uint32_t)std::max<int64_t>(a.n, 1); p.B = (uint32_t)a.B; p.A = a.A;
    p.mean = a.mean; p.log_std = a.log_std; p.actions = a.actions; p.old = a.log_pi_old;
    p.ref = a.log_pi_ref.p ? a.log_pi_ref : a.log_pi_old;
    p.own_ref = p.ref.p != p.old.p || p.ref.sb != p.old.sb || p.ref.sn != p.old.sn;
    p.adv = a.adv; p.mask = a.mask; p.moments = a.adv_moments;
    p.dlo = a.clip < 1.0 ? std::log1p(-a.clip) : -INFINITY; p.dhi = std::log1p(a.clip);       // (a ratio is never below 0)
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
    const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 1024);
    if (dtype == 0) hipLaunchKernelGGL(k_policy_loss_scale<float>, dim3(grid), dim3(256), 0, st, grad, n_mean, (float *)dmean, n_std, (float *)dlog_std);
    else hipLaunchKernelGGL(k_policy_loss_scale<bf16>, dim3(grid), dim3(256), 0, st, grad, n_mean, (bf16 *)dmean, n_std, (bf16 *)dlog_std);
    LAUNCH_CHECK();
    return 0;
}

int launch_gaussian_act(const ActArgs &a, hipStream_t st)
{
    const int64_t rows = a.B * a.n;
    if (rows == 0) return 0;
    const ActDev p{(uint32_t)rows, (uint32_t)a.n, a.A, a.mean, a.log_std, a.noise, a.actions, a.log_pi};
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
