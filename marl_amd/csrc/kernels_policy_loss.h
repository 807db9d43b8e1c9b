// The clipped policy loss of a diagonal Gaussian policy with its KL and entropy terms and its gradients, and the sampling
// of that policy.  Part of the translation unit seq_kernels.hip; not a stand-alone header.
//
// Row r (an agent at a step), action u, mean mu, s = log_std, z = (u - mu) e^-s:
//   log_pi = sum_j (-z_j^2 / 2 - s_j - log(2 pi) / 2)      d = log_pi - log_pi_old      q = e^d
//   L_r = -min(q A, clip(q, 1 - eps, 1 + eps) A) + kl (e^D - 1 - D) - ent H,   D = log_pi_ref - log_pi,  H = sum_j s_j + const
//   loss = mean of L_r over the rows the mask leaves (no rows: 0, and so are the gradients)
//   dL_r / dlog_pi = (cut ? 0 : -q A) - kl (e^D - 1),   cut = A > 0 and q > 1 + eps, or A < 0 and q < 1 - eps
//   dmu_j = dL/dlog_pi z_j e^-s_j,      ds_j = dL/dlog_pi (z_j^2 - 1) - ent
// The arithmetic of a row is in double: whether a ratio lies beyond the clipping border decides between a gradient and
// none, and e^D - 1 - D cancels for nearly equal policies (the CU's double rate equals its float rate, and the rows are
// bound by their bytes).  The gradients are written in the same pass as the loss: a mean over rows needs only their
// count, known without a mask and counted ahead with one.  Sums: per thread in double, per workgroup in a fixed order,
// then over the workgroups in a fixed order: the same inputs give the same bits.

constexpr int LOSS_SUMS = 5;                                            // gain, KL, entropy, cut rows, ratio; then A sums of ds

struct LossDev {
    int64_t rows, n, B;
    int A;
    Rows mean, log_std, actions, old, ref, adv, mask;
    const float *moments;
    double lo, hi, kl, ent;
    float *loss, *stats;
    void *dmean, *dstd;
    double *part;                                                       // [LOSS_SUMS + A][workgroups]
    const int64_t *counts;                                              // [workgroups] of the mask's count (several workgroups only)
    int n_counts;
};

template <int BS> __device__ __forceinline__ int64_t block_count(int64_t c, int64_t *sh)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = c;
    __syncthreads();
    int64_t t = 0;
    for (int w = 0; w < BS / 64; ++w) t += sh[w];
    return t;
}

// Valid rows of each workgroup's share, for a mask and several workgroups.
__global__ __launch_bounds__(256) void k_mask_count(int64_t rows, int64_t n, Rows mask, int64_t *counts)
{
    __shared__ int64_t sh[4];
    int64_t c = 0;
    const uint8_t *m = reinterpret_cast<const uint8_t *>(mask.p);
    for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < rows; r += (int64_t)gridDim.x * 256) {
        const int64_t b = r / n, i = r - b * n;
        c += m[b * mask.sb + i * mask.sn] != 0;
    }
    const int64_t t = block_count<256>(c, sh);
    if (threadIdx.x == 0) counts[blockIdx.x] = t;
}

template <typename TM, bool SHARED> __device__ __forceinline__ void loss_finish(const LossDev &p, const double *tot, int64_t count)
{
    if (threadIdx.x == 0) {
        const double inv = 1.0 / (double)(count > 0 ? count : 1);
        const double gain = tot[0] * inv, kl = tot[1] * inv, ent = tot[2] * inv;
        p.loss[0] = (float)(-gain + p.kl * kl - p.ent * ent);
        p.stats[0] = (float)gain; p.stats[1] = (float)kl; p.stats[2] = (float)ent;
        p.stats[3] = (float)(tot[3] * inv); p.stats[4] = (float)(tot[4] * inv); p.stats[5] = (float)count;
    }
    if (SHARED && threadIdx.x < (unsigned)p.A) reinterpret_cast<TM *>(p.dstd)[threadIdx.x] = from_float<TM>((float)tot[LOSS_SUMS + threadIdx.x]);
}

// A row is worked on by GL neighbouring lanes, AM components each (lane `sub` of them has components sub AM .. sub AM + AM - 1):
// one lane up to four components, more lanes beyond, so that no variant keeps more than four components' values in
// registers.  SHARED: one log_std for all rows.  PACKED: A == GL AM and the rows of mean (and log_std) are contiguous and
// aligned to AM values: one load each.
template <typename TM, int AM, int GL, bool SHARED, bool PACKED, int BS>
__global__ __launch_bounds__(BS) void k_policy_loss(LossDev p)
{
    constexpr int K = LOSS_SUMS + (SHARED ? AM * GL : 0), ROWS = BS / GL;
    __shared__ double sh_s[AM * GL], sh_e[AM * GL], red[BS / 64][K], tot[K];
    __shared__ int64_t sh_c[BS / 64];
    const int tid = threadIdx.x, sub = GL > 1 ? tid & (GL - 1) : 0, j0 = sub * AM;
    const bool masked = p.mask.p != nullptr;
    const uint8_t *maskp = reinterpret_cast<const uint8_t *>(p.mask.p);
    if (SHARED && tid < p.A) {
        const double s = (double)to_float(reinterpret_cast<const TM *>(p.log_std.p)[tid * p.log_std.sa]);
        sh_s[tid] = s; sh_e[tid] = exp(-s);
    }
    int64_t count = p.rows;
    if (masked) {
        int64_t c = 0;
        if (gridDim.x == 1) {
            for (int64_t r = tid; r < p.rows; r += BS) { const int64_t b = r / p.n, i = r - b * p.n; c += maskp[b * p.mask.sb + i * p.mask.sn] != 0; }
        } else {
            for (int k = tid; k < p.n_counts; k += BS) c += p.counts[k];
        }
        count = block_count<BS>(c, sh_c);
    }
    __syncthreads();
    const double w = 1.0 / (double)(count > 0 ? count : 1);
    double am = 0.0, ar = 1.0;
    if (p.moments) { am = (double)p.moments[0]; ar = (double)p.moments[1]; }
    double sum[LOSS_SUMS + AM];
#pragma unroll
    for (int k = 0; k < LOSS_SUMS + AM; ++k) sum[k] = 0.0;

    // The element offsets of a thread's row in each tensor move on by additions: the division and the products of an
    // address are paid once per thread.
    const int64_t stride = (int64_t)gridDim.x * ROWS, db = stride / p.n, di = stride - db * p.n;
    int64_t r = (int64_t)blockIdx.x * ROWS + tid / GL, b0 = r / p.n, i = r - b0 * p.n;
    int64_t o_mean = b0 * p.mean.sb + i * p.mean.sn + j0 * p.mean.sa, o_act = b0 * p.actions.sb + i * p.actions.sn + j0 * p.actions.sa,
            o_old = b0 * p.old.sb + i * p.old.sn, o_ref = b0 * p.ref.sb + i * p.ref.sn, o_adv = b0 * p.adv.sb + i * p.adv.sn,
            o_mask = b0 * p.mask.sb + i * p.mask.sn, o_std = b0 * p.log_std.sb + i * p.log_std.sn + j0 * p.log_std.sa;
    // (the GL lanes of a row leave the loop together)
    for (; r < p.rows; r += stride) {
        const bool valid = !masked || maskp[o_mask] != 0;
        float mu[AM], u[AM], sd[AM];
        if (PACKED) {
            load_vec<TM, AM>(mu, p.mean.p, o_mean);
            if (!SHARED) load_vec<TM, AM>(sd, p.log_std.p, o_std);
        }
#pragma unroll
        for (int j = 0; j < AM; ++j) {
            const bool has = PACKED || j0 + j < p.A;
            if (!PACKED) {
                mu[j] = has ? to_float(reinterpret_cast<const TM *>(p.mean.p)[o_mean + j * p.mean.sa]) : 0.f;
                if (!SHARED) sd[j] = has ? to_float(reinterpret_cast<const TM *>(p.log_std.p)[o_std + j * p.log_std.sa]) : 0.f;
            }
            u[j] = has ? reinterpret_cast<const float *>(p.actions.p)[o_act + j * p.actions.sa] : 0.f;
        }
        const double old = (double)reinterpret_cast<const float *>(p.old.p)[o_old];
        const double ref = (double)reinterpret_cast<const float *>(p.ref.p)[o_ref];
        const double adv = ((double)reinterpret_cast<const float *>(p.adv.p)[o_adv] - am) * ar;

        double z[AM], e[AM], lp = 0.0, ent = 0.0;
#pragma unroll
        for (int j = 0; j < AM; ++j) {
            if (PACKED || j0 + j < p.A) {
                const double s = SHARED ? sh_s[j0 + j] : (double)sd[j];
                e[j] = SHARED ? sh_e[j0 + j] : exp(-s);
                z[j] = ((double)u[j] - (double)mu[j]) * e[j];
                lp -= 0.5 * z[j] * z[j] + s + 0.91893853320467274178;   // log(2 pi) / 2
                ent += s + 1.41893853320467274178;                      // (log(2 pi) + 1) / 2
            }
        }
#pragma unroll
        for (int o = GL / 2; o; o >>= 1) { lp += __shfl_xor(lp, o, 64); ent += __shfl_xor(ent, o, 64); }
        const double q = exp(lp - old), D = ref - lp, em = expm1(D);
        const bool cut = (adv > 0.0 && q > p.hi) || (adv < 0.0 && q < p.lo);
        const double g = valid ? w * ((cut ? 0.0 : -q * adv) - p.kl * em) : 0.0;
        const double qa = q * adv, qc = (q < p.lo ? p.lo : q > p.hi ? p.hi : q) * adv;
        if (valid && sub == 0) {
            sum[0] += qa < qc ? qa : qc + (qa - qa);                     // min, and a NaN of either
            sum[1] += em - D;
            sum[2] += ent;
            sum[3] += cut ? 1.0 : 0.0;
            sum[4] += q;
        }
        float dm[AM], ds[AM];
#pragma unroll
        for (int j = 0; j < AM; ++j) {
            dm[j] = 0.f; ds[j] = 0.f;
            if (PACKED || j0 + j < p.A) {
                const double dsj = valid ? g * (z[j] * z[j] - 1.0) - p.ent * w : 0.0;
                dm[j] = valid ? (float)(g * z[j] * e[j]) : 0.f;
                if constexpr (SHARED) sum[LOSS_SUMS + j] += dsj;
                else ds[j] = (float)dsj;
            }
        }
        const int64_t at = r * p.A + j0;
        if (PACKED) {
            store_vec<TM, AM>(p.dmean, at, dm);
            if (!SHARED) store_vec<TM, AM>(p.dstd, at, ds);
        } else {
#pragma unroll
            for (int j = 0; j < AM; ++j)
                if (j0 + j < p.A) {
                    reinterpret_cast<TM *>(p.dmean)[at + j] = from_float<TM>(dm[j]);
                    if (!SHARED) reinterpret_cast<TM *>(p.dstd)[at + j] = from_float<TM>(ds[j]);
                }
        }
        i += di;
        const bool nb = i >= p.n;
        if (nb) i -= p.n;
        auto move = [&](int64_t &o, const Rows &t) __attribute__((always_inline)) { o += db * t.sb + di * t.sn; if (nb) o += t.sb - p.n * t.sn; };
        move(o_mean, p.mean); move(o_act, p.actions); move(o_old, p.old); move(o_ref, p.ref); move(o_adv, p.adv);
        if (masked) move(o_mask, p.mask);
        if (!SHARED) move(o_std, p.log_std);
    }
#pragma unroll
    for (int k = 0; k < LOSS_SUMS; ++k) {
        const double t = wave_sum(sum[k]);
        if ((tid & 63) == 0) red[tid >> 6][k] = t;
    }
    if constexpr (SHARED) {
#pragma unroll
        for (int j = 0; j < AM; ++j) {
            double t = sum[LOSS_SUMS + j];
#pragma unroll
            for (int o = 32; o >= GL; o >>= 1) t += __shfl_xor(t, o, 64);
            if ((tid & 63) < GL) red[tid >> 6][LOSS_SUMS + j0 + j] = t;
        }
    }
    __syncthreads();
    const int keys = LOSS_SUMS + (SHARED ? p.A : 0);
    if (tid < keys) {
        double t = 0.0;
        for (int v = 0; v < BS / 64; ++v) t += red[v][tid];
        if (gridDim.x == 1) tot[tid] = t;
        else p.part[(int64_t)tid * gridDim.x + blockIdx.x] = t;
    }
    if (gridDim.x == 1) {
        __syncthreads();
        loss_finish<TM, SHARED>(p, tot, count);
    }
}

// The workgroups' partial sums in a fixed order: a wave for each sum.
template <typename TM, bool SHARED> __global__ __launch_bounds__(512) void k_policy_loss_finish(LossDev p, int groups)
{
    __shared__ double tot[LOSS_SUMS + 32];
    __shared__ int64_t sh_c[8];
    int64_t count = p.rows;
    if (p.mask.p) {
        int64_t c = 0;
        for (int k = threadIdx.x; k < p.n_counts; k += 512) c += p.counts[k];
        count = block_count<512>(c, sh_c);
    }
    const int keys = LOSS_SUMS + (SHARED ? p.A : 0);
    for (int k = threadIdx.x >> 6; k < keys; k += 8) {
        double t = 0.0;
        for (int g = threadIdx.x & 63; g < groups; g += 64) t += p.part[(int64_t)k * groups + g];
        t = wave_sum(t);
        if ((threadIdx.x & 63) == 0) tot[k] = t;
    }
    __syncthreads();
    loss_finish<TM, SHARED>(p, tot, count);
}

// The gradients were written for an upstream gradient of 1; nothing is read or written when it is that.
template <typename TM> __global__ __launch_bounds__(256) void k_policy_loss_scale(const float *grad, int64_t n0, TM *g0, int64_t n1, TM *g1)
{
    const float s = grad[0];
    if (s == 1.0f) return;
    for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < n0 + n1; k += (int64_t)gridDim.x * 256) {
        TM *q = k < n0 ? g0 + k : g1 + (k - n0);
        *q = from_float<TM>(to_float(*q) * s);
    }
}

struct ActDev { int64_t rows, n; int A, shared; Rows mean, log_std, noise, actions, log_pi; };

// u = mu + e^s noise (or the given u), and the log-probability of u as it is stored.
template <typename TM, bool DRAW> __global__ __launch_bounds__(256) void k_gaussian_act(ActDev p)
{
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= p.rows) return;
    const int64_t b = r / p.n, i = r - b * p.n;
    const TM *mean = reinterpret_cast<const TM *>(p.mean.p) + b * p.mean.sb + i * p.mean.sn;
    const TM *std_ = reinterpret_cast<const TM *>(p.log_std.p) + b * p.log_std.sb + i * p.log_std.sn;
    const float *noise = DRAW ? reinterpret_cast<const float *>(p.noise.p) + b * p.noise.sb + i * p.noise.sn : nullptr;
    float *act = reinterpret_cast<float *>(const_cast<void *>(p.actions.p)) + b * p.actions.sb + i * p.actions.sn;
    double lp = 0.0;
    for (int j = 0; j < p.A; ++j) {
        const double mu = (double)to_float(mean[j * p.mean.sa]), s = (double)to_float(std_[j * p.log_std.sa]);
        float u;
        if (DRAW) {
            u = (float)(mu + exp(s) * (double)noise[j * p.noise.sa]);
            act[j * p.actions.sa] = u;
        } else {
            u = act[j * p.actions.sa];
        }
        const double z = ((double)u - mu) * exp(-s);
        lp -= 0.5 * z * z + s + 0.91893853320467274178;
    }
    reinterpret_cast<float *>(const_cast<void *>(p.log_pi.p))[b * p.log_pi.sb + i * p.log_pi.sn] = (float)lp;
}
