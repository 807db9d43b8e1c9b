// First-order recurrences over time: the gated memory of a policy (forward and backward) and the advantages of an episode.
// Part of the translation unit seq_kernels.hip (included there, inside namespace asmseq); not a stand-alone header.
//
// Every one of them is a chain of affine maps y_t = A_t y_{t-1} + S_t, independent for each channel, and two affine maps
// compose to an affine map, so any stretch of time can be summed up as one pair (A, S) before the state that enters it is
// known:
//   memory, forward     a = sigmoid(gate_t), h_t = a h_{t-1} + (1 - a) x_t                 A = a, S = (1 - a) x
//   memory, backward    G_t = dh_t + c_{t+1} (the gradient of h_t), c_t = a G_t, time reversed   A = a, S = a dh
//                       dx = (1 - a) G, dgate = G (h_{t-1} - x_t) a (1 - a), dh0 = c_0
//   advantages          delta = r + gamma (1 - done) V_{t+1} - V_t, time reversed          A = gamma lambda (1 - done), S = delta
// A step at which the state is dropped (a reset, a finished episode) is A = -0.0: no product of the other coefficients,
// which are never negative, has a sign, so the sign bit says "cut" through any composition and the state behind it is
// selected away rather than multiplied by zero (it may be infinite or NaN).  A step beyond a sequence's length is the
// identity (A = 1, S = 0).
//
// Work split: a workgroup takes 64 V neighbouring channels (V a lane) and walks its stretch of time in tiles of NW x L
// steps: wave w loads steps w L .. w L + L - 1 of the tile into registers, every load in flight at once, composes them,
// leaves the pair in LDS, and behind one barrier composes the pairs of the waves in front of it and walks its own steps
// again from registers.  Inputs are read once, outputs written once.  Where the channels alone do not fill the chip,
// the time axis is cut into `nsplit` stretches: a first launch composes each stretch (its reads leave the data in the
// last-level cache for the second), the second one starts each stretch from the composition of those before it.

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

template <typename T, int V> __device__ __forceinline__ void load_vec(float (&o)[V], const void *p, int64_t off)
{
    const Pack<T, V> r = *reinterpret_cast<const Pack<T, V> *>(reinterpret_cast<const T *>(p) + off);
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = to_float(r.v[v]);
}
template <typename T, int V> __device__ __forceinline__ void store_vec(void *p, int64_t off, const float (&x)[V])
{
    Pack<T, V> r;
#pragma unroll
    for (int v = 0; v < V; ++v) r.v[v] = from_float<T>(x[v]);
    *reinterpret_cast<Pack<T, V> *>(reinterpret_cast<T *>(p) + off) = r;
}

constexpr float CUT = -0.0f;
__device__ __forceinline__ float apply(float A, float S, float y) { return (__float_as_uint(A) >> 31) ? S : __fmaf_rn(A, y, S); }

// a = sigmoid(g), b = 1 - a, both to a few ulps at either end: the exponential of the negative magnitude never overflows
// and the smaller of the two is e / (1 + e) itself.
__device__ __forceinline__ void gate_pair(float g, float &a, float &b)
{
    const float e = expf(-fabsf(g)), p = 1.0f / (1.0f + e), q = e * p;
    a = g >= 0.f ? p : q;
    b = g >= 0.f ? q : p;
}

struct ScanGeom {
    int T, nsplit, Ts;              // steps, stretches, steps of a stretch (a multiple of the tile)
    int64_t C;                      // channels
    int64_t D;                      // channels of a sequence
    float *ws;                      // [nsplit][2][C]: the composition of each stretch
};

// What cuts and ends the sequences of a memory (MSK: any of it given).
struct Marks {
    const int *lengths;
    const uint8_t *resets;
    int64_t r_st, r_sb;
};
struct MarkLane { int len; int64_t r; };
__device__ __forceinline__ MarkLane mark_lane(const Marks &m, int64_t b, int T)
{
    int len = T;
    if (m.lengths) { len = m.lengths[b]; len = len < 0 ? 0 : len > T ? T : len; }
    return {len, b * m.r_sb};
}

// ---- the operators: load() fetches step t of this lane's channels, coef() turns it into its map, step() applies it and
// writes the step's outputs.  `on` is false beyond the stretch's end (the map is then the identity, nothing is written).

template <typename T, int V, bool MSK> struct ForwardOp {
    static constexpr bool REVERSE = false, SUMS = false, MOMENTS = false;
    Seq gate, x;
    SeqOut out;
    const float *h0;
    float *h_last;
    Marks marks;
    struct Lane { int64_t g, x, o; MarkLane m; };
    struct Item { float A[V], S[V]; uint8_t cut; };
    __device__ Lane lane(const ScanGeom &q, int64_t ch) const
    {
        const int64_t b = ch / q.D, d = ch - b * q.D;
        Lane l{b * gate.sb + d, b * x.sb + d, b * out.sb + d, {}};
        if (MSK) l.m = mark_lane(marks, b, q.T);
        return l;
    }
    __device__ void carry0(float (&c)[V], int64_t ch) const
    {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = 0.f;
        if (h0) load_vec<float, V>(c, h0, ch);
    }
    __device__ void load(Item &i, const Lane &l, int t, bool) const
    {
        load_vec<T, V>(i.A, gate.p, l.g + (int64_t)t * gate.st);
        load_vec<T, V>(i.S, x.p, l.x + (int64_t)t * x.st);
        if (MSK) i.cut = marks.resets ? marks.resets[l.m.r + (int64_t)t * marks.r_st] : 0;
    }
    __device__ void coef(Item &i, const Lane &l, int t, bool on) const
    {
        if (MSK) on = on && t < l.m.len;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float a, b;
            gate_pair(i.A[v], a, b);
            if (MSK && i.cut) a = CUT;
            i.S[v] = on ? b * i.S[v] : 0.f;
            i.A[v] = on ? a : 1.f;
        }
    }
    __device__ void step(float (&c)[V], const Item &i, const Lane &l, int t, bool on) const
    {
        float o[V];
        const bool in = !MSK || t < l.m.len;
#pragma unroll
        for (int v = 0; v < V; ++v) { c[v] = apply(i.A[v], i.S[v], c[v]); o[v] = in ? c[v] : 0.f; }
        if (on) store_vec<T, V>(out.p, l.o + (int64_t)t * out.st, o);
    }
    __device__ void finish(const float (&c)[V], int64_t ch) const { if (h_last) store_vec<float, V>(h_last, ch, c); }
};

template <typename T, int V, bool MSK> struct BackwardOp {
    static constexpr bool REVERSE = true, SUMS = false, MOMENTS = false;
    Seq gate, x, h, dh;
    SeqOut dgate, dx;
    const float *h0, *dh_last;
    float *dh0;
    Marks marks;
    struct Lane { int64_t g, x, h, dh, dg, dx, ch; MarkLane m; };
    struct Item { float A[V], S[V], b[V], m[V], dh[V]; uint8_t cut; };
    __device__ Lane lane(const ScanGeom &q, int64_t ch) const
    {
        const int64_t b = ch / q.D, d = ch - b * q.D;
        Lane l{b * gate.sb + d, b * x.sb + d, b * h.sb + d, b * dh.sb + d, b * dgate.sb + d, b * dx.sb + d, ch, {}};
        if (MSK) l.m = mark_lane(marks, b, q.T);
        return l;
    }
    __device__ void carry0(float (&c)[V], int64_t ch) const
    {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = 0.f;
        if (dh_last) load_vec<float, V>(c, dh_last, ch);
    }
    // agg: only what the composition needs
    __device__ void load(Item &i, const Lane &l, int t, bool agg) const
    {
        load_vec<T, V>(i.A, gate.p, l.g + (int64_t)t * gate.st);
        if (dh.p) load_vec<T, V>(i.dh, dh.p, l.dh + (int64_t)t * dh.st);
        if (MSK) i.cut = marks.resets ? marks.resets[l.m.r + (int64_t)t * marks.r_st] : 0;
        if (!agg) {
            load_vec<T, V>(i.b, x.p, l.x + (int64_t)t * x.st);
            load_vec<T, V>(i.m, h.p, l.h + (int64_t)(t > 0 ? t - 1 : 0) * h.st);
            if (t == 0) {
#pragma unroll
                for (int v = 0; v < V; ++v) i.m[v] = 0.f;
                if (h0) load_vec<float, V>(i.m, h0, l.ch);
            }
        }
    }
    __device__ void coef(Item &i, const Lane &l, int t, bool on) const
    {
        if (MSK) on = on && t < l.m.len;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float a, b;
            gate_pair(i.A[v], a, b);
            const float dh_v = dh.p ? i.dh[v] : 0.f, before = (MSK && i.cut) ? 0.f : i.m[v];
            i.m[v] = (before - i.b[v]) * a;                              // (h_{t-1} - x_t) a; x was loaded into b
            i.b[v] = b;
            i.dh[v] = dh_v;
            i.S[v] = on ? a * dh_v : 0.f;
            if (MSK && i.cut) { a = CUT; i.S[v] = 0.f; }
            i.A[v] = on ? a : 1.f;
        }
    }
    __device__ void step(float (&c)[V], const Item &i, const Lane &l, int t, bool on) const
    {
        float og[V], ox[V];
        const bool in = !MSK || t < l.m.len;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float G = (i.dh[v] + c[v]) * i.b[v];
            ox[v] = in ? G : 0.f;
            og[v] = in ? G * i.m[v] : 0.f;
            c[v] = apply(i.A[v], i.S[v], c[v]);
        }
        if (on) {
            store_vec<T, V>(dgate.p, l.dg + (int64_t)t * dgate.st, og);
            store_vec<T, V>(dx.p, l.dx + (int64_t)t * dx.st, ox);
        }
    }
    __device__ void finish(const float (&c)[V], int64_t ch) const { if (dh0) store_vec<float, V>(dh0, ch, c); }
};

// MSK: lengths or dones given.  Rows of one time step are contiguous (C channels), lengths belong to D channels each.
template <int V, bool MSK, bool MOM> struct AdvantageOp {
    static constexpr bool REVERSE = true, SUMS = true, MOMENTS = MOM;
    const float *rewards, *values;
    int64_t rew_st, val_st, done_st;
    const uint8_t *dones;
    const int *lengths;
    float gamma, lam;
    float *adv, *ret;
    int64_t C;
    struct Lane { int64_t ch; int len[V]; };
    struct Item { float A[V], S[V], val[V]; Pack<uint8_t, V> cut; };
    __device__ Lane lane(const ScanGeom &q, int64_t ch) const
    {
        Lane l{ch, {}};
        if (MSK) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                int n = q.T;
                if (lengths) { n = lengths[(ch + v) / q.D]; n = n < 0 ? 0 : n > q.T ? q.T : n; }
                l.len[v] = n;
            }
        }
        return l;
    }
    __device__ void carry0(float (&c)[V], int64_t) const
    {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = 0.f;
    }
    __device__ void load(Item &i, const Lane &l, int t, bool) const
    {
        load_vec<float, V>(i.S, rewards, l.ch + (int64_t)t * rew_st);
        load_vec<float, V>(i.val, values, l.ch + (int64_t)t * val_st);
        load_vec<float, V>(i.A, values, l.ch + (int64_t)(t + 1) * val_st);
        if (MSK && dones) i.cut = *reinterpret_cast<const Pack<uint8_t, V> *>(dones + l.ch + (int64_t)t * done_st);
    }
    __device__ void coef(Item &i, const Lane &l, int t, bool on) const
    {
        const float gl = gamma * lam;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const bool in = on && (!MSK || t < l.len[v]), cut = MSK && dones && i.cut.v[v];
            const float delta = i.S[v] + (cut ? 0.f : gamma * i.A[v]) - i.val[v];
            i.S[v] = in ? delta : 0.f;
            i.A[v] = in ? (cut ? CUT : gl) : 1.f;
        }
    }
    __device__ void step(float (&c)[V], const Item &i, const Lane &l, int t, bool on, double &s1, double &s2, int64_t &cnt) const
    {
        float oa[V], ov[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            c[v] = apply(i.A[v], i.S[v], c[v]);
            const bool in = on && (!MSK || t < l.len[v]);
            oa[v] = in ? c[v] : 0.f;
            ov[v] = in ? c[v] + i.val[v] : 0.f;
            if (MOM && in) { s1 += (double)c[v]; s2 += (double)c[v] * (double)c[v]; ++cnt; }
        }
        if (on) {
            store_vec<float, V>(adv, l.ch + (int64_t)t * C, oa);
            store_vec<float, V>(ret, l.ch + (int64_t)t * C, ov);
        }
    }
    __device__ void finish(const float (&)[V], int64_t) const {}
};

// Moments of the advantages: a partial (count, sum, sum of squares) per workgroup in double, summed in a fixed order.
__device__ __forceinline__ double wave_sum(double x)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// V channels a lane, NW waves, L steps a wave and tile.  AGG: the stretch's composition only.
template <class Op, int V, int NW, int L, bool AGG>
__global__ __launch_bounds__(64 * NW) void k_scan(Op op, ScanGeom q, double *mom)
{
    __shared__ alignas(16) float ex[2][NW][2][64][V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), split = blockIdx.y;
    const int64_t ch0 = ((int64_t)blockIdx.x * 64 + lane) * V;
    const bool have = ch0 < q.C;
    const int64_t ch = have ? ch0 : 0;                                  // (lanes beyond the channels read channel 0 and write nothing)
    const typename Op::Lane ln = op.lane(q, ch);
    const int lo = split * q.Ts, hi = lo + q.Ts < q.T ? lo + q.Ts : q.T;
    float CA[V], c[V];                                                  // AGG: (CA, c) is the composition so far; else c is the state
    if (AGG) {
#pragma unroll
        for (int v = 0; v < V; ++v) { CA[v] = 1.f; c[v] = 0.f; }
    } else {
        op.carry0(c, ch);
        for (int j = 0; j < split; ++j) {
            float A[V], S[V];
            load_vec<float, V>(A, q.ws, (int64_t)(2 * j) * q.C + ch);
            load_vec<float, V>(S, q.ws, (int64_t)(2 * j + 1) * q.C + ch);
#pragma unroll
            for (int v = 0; v < V; ++v) c[v] = apply(A[v], S[v], c[v]);
        }
    }
    double s1 = 0, s2 = 0;
    int64_t cnt = 0;
    int par = 0;
    for (int tile = lo; tile < hi; tile += NW * L) {
        const int u0 = tile + wave * L;
        typename Op::Item it[L];
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const int u = u0 + l < hi ? u0 + l : hi - 1;                // (steps beyond the end: the last one again, not used)
            op.load(it[l], ln, Op::REVERSE ? q.T - 1 - u : u, AGG);
        }
        float PA[V], PS[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { PA[v] = 1.f; PS[v] = 0.f; }
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const int u = u0 + l;
            op.coef(it[l], ln, Op::REVERSE ? q.T - 1 - u : u, u < hi);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                PS[v] = apply(it[l].A[v], it[l].S[v], PS[v]);
                PA[v] = (__float_as_uint(it[l].A[v]) >> 31) ? CUT : it[l].A[v] * PA[v];
            }
        }
        float mine[V];                                                  // the state in front of this wave's steps
        if (NW > 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) { ex[par][wave][0][lane][v] = PA[v]; ex[par][wave][1][lane][v] = PS[v]; }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                if (w == wave) {
#pragma unroll
                    for (int v = 0; v < V; ++v) mine[v] = c[v];
                }
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float A = ex[par][w][0][lane][v], S = ex[par][w][1][lane][v];
                    c[v] = apply(A, S, c[v]);
                    if (AGG) CA[v] = (__float_as_uint(A) >> 31) ? CUT : A * CA[v];
                }
            }
            par ^= 1;                                                   // (the next tile's pairs go to the other half: one barrier a tile)
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                mine[v] = c[v];
                if (AGG) { c[v] = apply(PA[v], PS[v], c[v]); CA[v] = (__float_as_uint(PA[v]) >> 31) ? CUT : PA[v] * CA[v]; }
            }
        }
        if (!AGG) {
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const int u = u0 + l, t = Op::REVERSE ? q.T - 1 - u : u;
                if constexpr (Op::SUMS) op.step(mine, it[l], ln, t, have && u < hi, s1, s2, cnt);
                else op.step(mine, it[l], ln, t, have && u < hi);
            }
            if (NW == 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) c[v] = mine[v];
            }
        }
    }
    if (AGG) {
        if (have && wave == 0) {
            store_vec<float, V>(q.ws, (int64_t)(2 * split) * q.C + ch, CA);
            store_vec<float, V>(q.ws, (int64_t)(2 * split + 1) * q.C + ch, c);
        }
        return;
    }
    if (have && wave == 0 && split == q.nsplit - 1) op.finish(c, ch);
    if constexpr (Op::MOMENTS) {
        __shared__ double red[NW][3];
        const double w1 = wave_sum(s1), w2 = wave_sum(s2), w0 = wave_sum((double)cnt);
        if (lane == 0) { red[wave][0] = w0; red[wave][1] = w1; red[wave][2] = w2; }
        __syncthreads();
        if (threadIdx.x < 3) {
            double t = 0;
            for (int w = 0; w < NW; ++w) t += red[w][threadIdx.x];
            mom[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 3 + threadIdx.x] = t;
        }
    }
}

// One workgroup: (mean, 1 / (standard deviation + 1e-8)) of the advantages from the partials of k_scan.
__global__ __launch_bounds__(256) void k_moments(const double *mom, int64_t n, float *out)
{
    __shared__ double red[4][3];
    double s[3] = {0, 0, 0};
    for (int64_t k = threadIdx.x; k < n; k += 256)
#pragma unroll
        for (int j = 0; j < 3; ++j) s[j] += mom[k * 3 + j];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
        const double t = wave_sum(s[j]);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][j] = t;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double t[3];
        for (int j = 0; j < 3; ++j) t[j] = red[0][j] + red[1][j] + red[2][j] + red[3][j];
        const double k = t[0] > 0 ? t[0] : 1.0, mean = t[1] / k, var = t[2] / k - mean * mean;
        out[0] = (float)mean;
        out[1] = (float)(1.0 / (sqrt(var > 0 ? var : 0.0) + 1e-8));
    }
}

// One step of the memory: state <- a k state + (1 - a) x, out = the new state in the inputs' type.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_scan_step(int64_t n, int64_t D, const void *gate, int64_t g_sb, const void *x, int64_t x_sb,
                                                   float *state, const uint8_t *reset, int64_t r_sb, void *out, int64_t o_sb)
{
    const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (e >= n) return;
    const int64_t b = e / D, d = e - b * D;
    float g[V], xv[V], s[V];
    load_vec<T, V>(g, gate, b * g_sb + d);
    load_vec<T, V>(xv, x, b * x_sb + d);
    load_vec<float, V>(s, state, e);
    const bool cut = reset && reset[b * r_sb];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float a, k;
        gate_pair(g[v], a, k);
        s[v] = apply(cut ? CUT : a, k * xv[v], s[v]);
    }
    store_vec<float, V>(state, e, s);
    store_vec<T, V>(out, b * o_sb + d, s);
}
