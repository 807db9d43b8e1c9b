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
// Where the state is dropped (a reset, a finished episode), A = 0 and the state is selected away rather than multiplied by
// it (it may be infinite or NaN).  The composition of a stretch that holds such a step has A = -0.0: coefficients are never
// negative, so the sign says it.  A step beyond a sequence's length is the identity (A = 1, S = 0).
//
// Work split: a workgroup takes 64 V neighbouring channels (V a lane) and walks its stretch of time in tiles of NW x L
// steps: wave w has steps w L .. w L + L - 1 of the tile in registers, composes them, leaves the pair in LDS, and behind one
// barrier composes the pairs of the waves in front of it and walks its own steps again from registers; the loads of its
// next tile are in flight meanwhile.  Inputs are read once, outputs written once.  Where the channels alone do not fill
// the chip, the time axis is cut into `nsplit` stretches: a first launch composes each stretch (its reads leave the data
// in the last-level cache for the second), the second one starts each stretch from the composition of those before it.
//
// Measured: 200 steps x 491520 channels of float32 forward 241 us for 1.23 GB (5.1 TB/s, what a copy reaches: bound by HBM), 200 x 62848
// of bfloat16 with resets and lengths forward 25 us for 83 MB (3.3 TB/s: 31 vector instructions an element and a step), backward 40 us
// for 133 MB (72 of them, 25 us of issue; two waves a SIMD cover the rest badly), 37 x 1920 3.9 us (a launch and two trips to memory).
//
// Addresses: a tensor's base at this step and at the workgroup's first sequence is uniform (scalar registers), a lane adds a
// 32-bit byte offset (OFF = uint32_t), or a 64-bit one where a workgroup's sequences lie too far apart (OFF = int64_t).

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

// The [B][D] arrays in front of and behind a sequence, of any alignment (read and written once).
template <int V> __device__ __forceinline__ void load_each(float (&o)[V], const float *p, uint32_t ch)
{
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = p ? p[ch + v] : 0.f;
}
template <int V> __device__ __forceinline__ void store_each(float *p, uint32_t ch, const float (&x)[V])
{
    if (p) {
#pragma unroll
        for (int v = 0; v < V; ++v) p[ch + v] = x[v];
    }
}

// a = sigmoid(g) and b = 1 - a from t = e^-|g| <= 1: the larger of the two is 1 / (1 + t), the smaller t / (1 + t), so neither end loses
// digits and nothing overflows.  |g| log2(e) = n + f with |f| <= 1/2, f by two fused products with the two parts of log2(e), so its
// rounding does not grow with |g|; 2^f and the reciprocal are the hardware's (1 unit in the last place each), the reciprocal
// with a Newton step.  a and b are good to 6 halves of a unit down to the smallest numbers.  n stops at 160, where t is 0.
// NaN stays NaN.
__device__ __forceinline__ void gate_pair(float g, float &a, float &b)
{
    const float y = fabsf(g);
    const float n = fmaxf(__builtin_rintf(y * -1.44269504088896340736f), -160.0f);
    const float f = __fmaf_rn(y, -1.92596299112661746887e-8f, __fmaf_rn(y, -1.44269504088896340736f, -n));
    const float t = __builtin_ldexpf(__builtin_amdgcn_exp2f(f), (int)n), s = 1.0f + t, r = __builtin_amdgcn_rcpf(s);
    const float big = __fmaf_rn(__fmaf_rn(-s, r, 1.0f), r, r), small = t * big;
    a = g < 0.0f ? small : big;
    b = g < 0.0f ? big : small;
}

struct ScanGeom {
    int T, nsplit, Ts;              // steps, stretches, steps of a stretch (a multiple of the tile)
    uint32_t C;                     // channels
    uint32_t D;                     // channels of a sequence
    float *ws;                      // [nsplit][C][2]: the composition (A, S) of each stretch
};

// Where a lane is: its channel, its sequence's distance from the workgroup's first one and its place in the sequence.
struct Place { uint32_t ch, b0, db, d; };

// What cuts and ends the sequences of a memory (MSK: any of it given).
struct Marks {
    const int *lengths;
    const uint8_t *resets;
    int64_t r_st, r_sb;
};
template <typename OFF> struct MarkLane { int len; OFF r; };
template <typename OFF> __device__ __forceinline__ MarkLane<OFF> mark_lane(const Marks &m, const Place &w, int T)
{
    int len = T;
    if (m.lengths) { len = m.lengths[(size_t)w.b0 + w.db]; len = len < 0 ? 0 : len > T ? T : len; }
    return {len, (OFF)((int64_t)w.db * m.r_sb)};
}

template <typename T, typename S> __device__ __forceinline__ const char *base_of(const S &s, uint32_t b0) { return reinterpret_cast<const char *>(s.p) + (int64_t)b0 * s.sb * (int64_t)sizeof(T); }
template <typename T, typename OFF, typename S> __device__ __forceinline__ OFF off_of(const S &s, const Place &w) { return (OFF)(((int64_t)w.db * s.sb + w.d) * (int64_t)sizeof(T)); }
// V values as they lie in memory, in 32-bit words: a load in flight is not waited for by an unpacking the compiler moved
// up to it.
template <typename T, int V> struct Words;
template <int V> struct Words<float, V> {
    Pack<float, V> w;
    __device__ __forceinline__ float get(int v) const { return w.v[v]; }
    __device__ __forceinline__ void load(const char *p) { w = *reinterpret_cast<const Pack<float, V> *>(p); }
};
template <int V> struct Words<bf16, V> {
    Pack<uint32_t, (V + 1) / 2> w;
    __device__ __forceinline__ float get(int v) const { return __uint_as_float(v & 1 ? w.v[v / 2] & 0xffff0000u : w.v[v / 2] << 16); }
    __device__ __forceinline__ void load(const char *p)
    {
        if constexpr (V == 1) w.v[0] = *reinterpret_cast<const uint16_t *>(p);
        else w = *reinterpret_cast<const Pack<uint32_t, V / 2> *>(p);
    }
};
template <int V> struct Words<uint8_t, V> {
    uint32_t w;
    __device__ __forceinline__ bool get(int v) const { return (w >> (8 * v)) & 0xffu; }
    __device__ __forceinline__ void load(const char *p)
    {
        if constexpr (V == 1) w = *reinterpret_cast<const uint8_t *>(p);
        else if constexpr (V == 2) w = *reinterpret_cast<const uint16_t *>(p);
        else w = *reinterpret_cast<const uint32_t *>(p);
    }
};
// A step is tb + dl with dl a constant of the unrolled loop: its offset is one product a tile and additions.
struct Step { int tb, dl; __device__ __forceinline__ int t() const { return tb + dl; } };
__device__ __forceinline__ int64_t step_off(const Step &s, int64_t st) { return (int64_t)s.tb * st + (int64_t)s.dl * st; }
template <typename T, int V, typename OFF> __device__ __forceinline__ void fetch(Words<T, V> &o, const char *base, int64_t step, OFF off)
{
    o.load(base + step * (int64_t)sizeof(T) + off);
}
template <typename T, int V, typename OFF> __device__ __forceinline__ void put(const char *base, int64_t step, OFF off, const float (&x)[V])
{
    Pack<T, V> r;
#pragma unroll
    for (int v = 0; v < V; ++v) r.v[v] = from_float<T>(x[v]);
    *reinterpret_cast<Pack<T, V> *>(const_cast<char *>(base) + step * (int64_t)sizeof(T) + off) = r;
}

// ---- the operators: fetch() loads step t of this lane's channels as it lies in memory, coef() turns it into its map, step()
// applies it and writes the step's outputs.  `on` is false beyond the stretch's end (the map is then the identity, nothing
// is written).

template <typename T, int V, bool MSK, typename OFF> struct ForwardOp {
    static constexpr bool REVERSE = false, SUMS = false, MOMENTS = false, CUTS = MSK, KEEPS = true, BLOCK = false;
    Seq gate, x;
    SeqOut out;
    const float *h0;
    float *h_last;
    float *ck;                                                          // (nullable) the state in front of step T - 8 (k + 1), at [k][channel]
    Marks marks;
    struct Lane { const char *g, *x, *o, *r; OFF og, ox, oo; MarkLane<OFF> m; };
    struct Raw { Words<T, V> g, x; Words<uint8_t, 1> cut; };
    struct Item { float A[V], S[V]; bool cut; };
    __device__ Lane lane(const ScanGeom &q, const Place &w) const
    {
        Lane l{base_of<T>(gate, w.b0), base_of<T>(x, w.b0), base_of<T>(out, w.b0), reinterpret_cast<const char *>(marks.resets) + (int64_t)w.b0 * marks.r_sb,
               off_of<T, OFF>(gate, w), off_of<T, OFF>(x, w), off_of<T, OFF>(out, w), {}};
        if (MSK) l.m = mark_lane<OFF>(marks, w, q.T);
        return l;
    }
    ForwardOp composing() const { return *this; }                       // (the operator of a launch that only composes)
    __device__ void carry0(float (&c)[V], uint32_t ch) const { load_each(c, h0, ch); }
    __device__ void load(Raw &i, const Lane &l, const Step &s, bool) const
    {
        fetch(i.g, l.g, step_off(s, gate.st), l.og);
        fetch(i.x, l.x, step_off(s, x.st), l.ox);
        if (MSK) { i.cut.w = 0; if (marks.resets) fetch(i.cut, l.r, step_off(s, marks.r_st), l.m.r); }
    }
    __device__ void coef(Item &o, const Raw &i, const Lane &l, const Step &s, bool on) const
    {
        if (MSK) on = on && s.t() < l.m.len;
        o.cut = MSK && on && i.cut.get(0);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float a, b;
            gate_pair(i.g.get(v), a, b);
            if (MSK && o.cut) a = 0.f;
            o.S[v] = on ? b * i.x.get(v) : 0.f;
            o.A[v] = on ? a : 1.f;
        }
    }
    __device__ void step(float (&c)[V], const Item &i, const Lane &l, const Step &s, bool on) const
    {
        float o[V];
        const bool in = !MSK || s.t() < l.m.len;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            c[v] = __fmaf_rn(i.A[v], MSK && i.cut ? 0.f : c[v], i.S[v]);
            o[v] = in ? c[v] : 0.f;
        }
        if (on) put<T, V>(l.o, step_off(s, out.st), l.oo, o);
    }
    __device__ void finish(const float (&c)[V], uint32_t ch) const { store_each(h_last, ch, c); }
};

// KEPT: the states in front of a wave's eight steps come from what the forward pass kept and are computed again in between, in
// float32, from the gates and inputs the pass reads anyway; else they are h as it is stored.  h in bfloat16 would give the
// gate's gradient, a product with h_{t-1} - x_t, an error of half a step of h: as much as the difference itself where the
// memory has settled near its input.
template <typename T, int V, bool MSK, typename OFF, bool KEPT> struct BackwardAnyOp {
    static constexpr bool REVERSE = true, SUMS = false, MOMENTS = false, CUTS = MSK, KEEPS = false, BLOCK = KEPT;
    Seq gate, x, h, dh;
    SeqOut dgate, dx;
    const float *h0, *dh_last;
    float *dh0;
    const float *ck;
    Marks marks;
    struct Lane { const char *g, *x, *h, *dh, *dg, *dx, *r; OFF og, ox, oh, odh, odg, odx; uint32_t ch; MarkLane<OFF> m; };
    struct Raw { Words<T, V> g, x, h, dh; Words<uint8_t, 1> cut; };
    struct Item { float A[V], S[V], b[V], m[V], dh[V]; bool cut; };
    __device__ Lane lane(const ScanGeom &q, const Place &w) const
    {
        Lane l{base_of<T>(gate, w.b0), base_of<T>(x, w.b0), base_of<T>(h, w.b0), base_of<T>(dh, w.b0), base_of<T>(dgate, w.b0), base_of<T>(dx, w.b0),
               reinterpret_cast<const char *>(marks.resets) + (int64_t)w.b0 * marks.r_sb, off_of<T, OFF>(gate, w), off_of<T, OFF>(x, w), off_of<T, OFF>(h, w),
               off_of<T, OFF>(dh, w), off_of<T, OFF>(dgate, w), off_of<T, OFF>(dx, w), w.ch, {}};
        if (MSK) l.m = mark_lane<OFF>(marks, w, q.T);
        return l;
    }
    BackwardAnyOp<T, V, MSK, OFF, false> composing() const { return {gate, x, h, dh, dgate, dx, h0, dh_last, dh0, ck, marks}; }      // (needs no states)
    __device__ void carry0(float (&c)[V], uint32_t ch) const { load_each(c, dh_last, ch); }
    // agg: only what the composition needs
    __device__ void load(Raw &i, const Lane &l, const Step &s, bool agg) const
    {
        fetch(i.g, l.g, step_off(s, gate.st), l.og);
        if (dh.p) fetch(i.dh, l.dh, step_off(s, dh.st), l.odh);
        if (MSK) { i.cut.w = 0; if (marks.resets) fetch(i.cut, l.r, step_off(s, marks.r_st), l.m.r); }
        if (!agg) {
            fetch(i.x, l.x, step_off(s, x.st), l.ox);
            if (!KEPT) fetch(i.h, l.h, s.t() > 0 ? step_off(Step{s.tb, s.dl - 1}, h.st) : 0, l.oh);
        }
    }
    // The state in front of the eight steps u0 .. u0 + 7 from the end (uniform).
    __device__ void load_state(float (&o)[V], const ScanGeom &q, int u0, uint32_t ch) const
    {
        if (u0 + 8 <= q.T) load_vec<float, V>(o, ck, (int64_t)(u0 / 8) * q.C + ch);
        else load_each(o, h0, ch);                                      // (the block that reaches the first step)
    }
    // Forwards through the block, whose step k lies k in front of `last`; steps from `n` on lie in front of the first one.
    template <int L> __device__ void states(Item (&o)[L], const Raw (&raw)[L], const float (&state)[V], const Lane &l, int last, int n) const
    {
        float before[V];
#pragma unroll
        for (int v = 0; v < V; ++v) before[v] = state[v];
#pragma unroll
        for (int k = L - 1; k >= 0; --k) {
            const bool on = k < n && (!MSK || last - k < l.m.len), cut = MSK && raw[k].cut.get(0);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a, b;
                gate_pair(raw[k].g.get(v), a, b);
                const float from = cut ? 0.f : before[v], xv = raw[k].x.get(v);
                o[k].A[v] = a;
                o[k].b[v] = b;
                o[k].m[v] = (from - xv) * a;
                const float after = __fmaf_rn(a, from, b * xv);
                before[v] = on ? after : before[v];
            }
        }
    }
    __device__ void coef(Item &o, const Raw &i, const Lane &l, const Step &s, bool on) const
    {
        if constexpr (KEPT) {                                           // (states() has left a, b and m)
            if (MSK) on = on && s.t() < l.m.len;
            o.cut = MSK && on && i.cut.get(0);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float a = MSK && o.cut ? 0.f : o.A[v];
                o.dh[v] = dh.p ? i.dh.get(v) : 0.f;
                o.S[v] = on && !(MSK && o.cut) ? a * o.dh[v] : 0.f;
                o.A[v] = on ? a : 1.f;
            }
            return;
        }
        float before[V];
#pragma unroll
        for (int v = 0; v < V; ++v) before[v] = i.h.get(v);
        if (s.t() == 0) load_each(before, h0, l.ch);                     // (uniform)
        if (MSK) on = on && s.t() < l.m.len;
        o.cut = MSK && on && i.cut.get(0);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float a, b;
            gate_pair(i.g.get(v), a, b);
            const float d = dh.p ? i.dh.get(v) : 0.f;
            o.m[v] = ((MSK && o.cut ? 0.f : before[v]) - i.x.get(v)) * a;       // (h_{t-1} - x_t) a
            o.b[v] = b;
            o.dh[v] = d;
            if (MSK && o.cut) a = 0.f;
            o.S[v] = on && !(MSK && o.cut) ? a * d : 0.f;
            o.A[v] = on ? a : 1.f;
        }
    }
    __device__ void step(float (&c)[V], const Item &i, const Lane &l, const Step &s, bool on) const
    {
        float og[V], ox[V];
        const bool in = !MSK || s.t() < l.m.len;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float G = (i.dh[v] + c[v]) * i.b[v];
            ox[v] = in ? G : 0.f;
            og[v] = in ? G * i.m[v] : 0.f;
            c[v] = __fmaf_rn(i.A[v], MSK && i.cut ? 0.f : c[v], i.S[v]);
        }
        if (on) {
            put<T, V>(l.dg, step_off(s, dgate.st), l.odg, og);
            put<T, V>(l.dx, step_off(s, dx.st), l.odx, ox);
        }
    }
    __device__ void finish(const float (&c)[V], uint32_t ch) const { store_each(dh0, ch, c); }
};

template <typename T, int V, bool MSK, typename OFF> using BackwardOp = BackwardAnyOp<T, V, MSK, OFF, false>;
template <typename T, int V, bool MSK, typename OFF> using BackwardKeptOp = BackwardAnyOp<T, V, MSK, OFF, true>;

// Number, mean and sum of squared distances from the mean of some values, in double.  add(): distances from the first of them;
// join(): two sets' means differ by d, which adds d^2 n1 n2 / (n1 + n2) (Chan, Golub and LeVeque).  (A mean of squares less the square of
// the mean would leave a deviation of 1e-8 of the mean where all values are equal.)
struct Spread { double n, mean, m2; };
struct SpreadSum {
    double first = 0.0, s = 0.0, ss = 0.0;
    int n = 0;
    __device__ __forceinline__ void add(double x)
    {
        first = n ? first : x;
        const double d = x - first;
        s += d; ss = __fma_rn(d, d, ss); ++n;
    }
    __device__ Spread spread() const
    {
        if (!n) return {0.0, 0.0, 0.0};
        const double m = s / n;
        return {(double)n, first + m, ss - s * m > 0.0 || ss != ss ? ss - s * m : 0.0};
    }
};
__device__ __forceinline__ Spread join(const Spread &a, const Spread &b)
{
    const double n = a.n + b.n, d = b.mean - a.mean, w = n > 0.0 ? b.n / n : 0.0;
    if (a.n == 0.0) return b;
    return b.n == 0.0 ? a : Spread{n, a.mean + d * w, a.m2 + b.m2 + d * d * a.n * w};
}
__device__ __forceinline__ Spread wave_join(Spread x)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const Spread y{__shfl_xor(x.n, o, 64), __shfl_xor(x.mean, o, 64), __shfl_xor(x.m2, o, 64)};
        x = threadIdx.x & o ? join(y, x) : join(x, y);
    }
    return x;
}

// 200 x 122880: 78 us for 395 MB (5.1 TB/s, bound by HBM).
// MSK: lengths or dones given.  Rows of one time step are contiguous (C channels), lengths belong to D channels each.
template <int V, bool MSK, bool MOM> struct AdvantageOp {
    static constexpr bool REVERSE = true, SUMS = true, MOMENTS = MOM, CUTS = MSK, KEEPS = false, BLOCK = false;
    const float *rewards, *values;
    int64_t rew_st, val_st, done_st;
    const uint8_t *dones;
    const int *lengths;
    float gamma, lam;
    float *adv, *ret;
    int64_t C;
    struct Lane { uint32_t ch; int len[V]; };
    struct Raw { Words<float, V> r, v0, v1; Words<uint8_t, V> cut; };
    struct Item { float A[V], S[V], val[V]; bool cut[V]; };
    __device__ Lane lane(const ScanGeom &q, const Place &w) const
    {
        Lane l{w.ch, {}};
        if (MSK) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                int n = q.T;
                if (lengths) { n = lengths[(w.ch + v) / q.D]; n = n < 0 ? 0 : n > q.T ? q.T : n; }
                l.len[v] = n;
            }
        }
        return l;
    }
    AdvantageOp composing() const { return *this; }
    __device__ void carry0(float (&c)[V], int64_t) const
    {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = 0.f;
    }
    static __device__ const char *at(const void *p) { return reinterpret_cast<const char *>(p); }
    __device__ void load(Raw &i, const Lane &l, const Step &s, bool) const
    {
        fetch(i.r, at(rewards), step_off(s, rew_st), l.ch * 4u);
        fetch(i.v0, at(values), step_off(s, val_st), l.ch * 4u);
        fetch(i.v1, at(values), step_off(Step{s.tb, s.dl + 1}, val_st), l.ch * 4u);
        if (MSK && dones) fetch(i.cut, at(dones), step_off(s, done_st), l.ch);
    }
    __device__ void coef(Item &o, const Raw &i, const Lane &l, const Step &s, bool on) const
    {
        const float gl = gamma * lam;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const bool in = on && (!MSK || s.t() < l.len[v]), cut = MSK && dones && i.cut.get(v);
            const float delta = i.r.get(v) + (cut ? 0.f : gamma * i.v1.get(v)) - i.v0.get(v);
            o.cut[v] = in && cut;
            o.val[v] = i.v0.get(v);
            o.S[v] = in ? delta : 0.f;
            o.A[v] = in ? (cut ? 0.f : gl) : 1.f;
        }
    }
    __device__ void step(float (&c)[V], const Item &i, const Lane &l, const Step &s, bool on, SpreadSum &sum) const
    {
        float oa[V], ov[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            c[v] = __fmaf_rn(i.A[v], MSK && i.cut[v] ? 0.f : c[v], i.S[v]);
            const bool in = on && (!MSK || s.t() < l.len[v]);
            oa[v] = in ? c[v] : 0.f;
            ov[v] = in ? c[v] + i.val[v] : 0.f;
            if (MOM && in) sum.add((double)c[v]);
        }
        if (on) {
            put<float, V>(at(adv), step_off(s, C), l.ch * 4u, oa);
            put<float, V>(at(ret), step_off(s, C), l.ch * 4u, ov);
        }
    }
    __device__ void finish(const float (&)[V], int64_t) const {}
};

template <class Item> __device__ __forceinline__ bool cut_of(const Item &i, int v)
{
    if constexpr (std::is_array_v<decltype(i.cut)>) return i.cut[v];
    else return i.cut;
}

__device__ __forceinline__ double wave_sum(double x)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// y behind a stretch whose composition is (A, S)
template <bool CUTS> __device__ __forceinline__ float through(float A, float S, float y)
{
    const float r = __fmaf_rn(A, y, S);
    return CUTS && (__float_as_uint(A) >> 31) ? S : r;
}
template <bool CUTS> __device__ __forceinline__ float joined(float A, float A0) { return CUTS && (__float_as_uint(A) >> 31) ? -0.f : A * A0; }

// V channels a lane, NW waves, L steps a wave and tile.  AGG: the stretch's composition only.
template <class Op, int V, int NW, int L, bool AGG>
__global__ __launch_bounds__(64 * NW) void k_scan(Op op, ScanGeom q, double *mom)
{
    constexpr bool CUTS = Op::CUTS;
    __shared__ alignas(16) float ex[NW > 1 ? 2 : 1][NW][2][64][V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), split = blockIdx.y;
    const uint32_t first = blockIdx.x * 64u * V, mine_ch = first + lane * V;
    const bool have = mine_ch < q.C;
    Place w;
    w.ch = have ? mine_ch : first;                                      // (lanes beyond the channels read the workgroup's first one and write nothing)
    w.b0 = __builtin_amdgcn_readfirstlane(first / q.D);
    const uint32_t rel = w.ch - w.b0 * q.D;
    w.db = rel / q.D;
    w.d = rel - w.db * q.D;
    const typename Op::Lane ln = op.lane(q, w);
    const int lo = split * q.Ts, hi = lo + q.Ts < q.T ? lo + q.Ts : q.T;
    typename Op::Raw raw[L];
    float state[V];                                                     // BLOCK: the state in front of this wave's steps
    static_assert(!AGG || NW > 1, "a wave that has all of time to itself composes nothing");
    static_assert(!Op::BLOCK || L == 8, "states are kept in front of every eighth step");
    auto step_at = [&](int u0, int l) __attribute__((always_inline)) { return Op::REVERSE ? Step{q.T - 1 - u0, -l} : Step{u0, l}; };
    // CLAMP: a step beyond the end reads the last one again, and is not used
    auto load_tile = [&](auto clamp, int tile) __attribute__((always_inline)) {
        const int u0 = tile + wave * L;
#pragma unroll
        for (int l = 0; l < L; ++l) {
            if (decltype(clamp)::value) op.load(raw[l], ln, step_at(u0 + l < hi ? u0 + l : hi - 1, 0), AGG);
            else op.load(raw[l], ln, step_at(u0, l), AGG);
        }
        if constexpr (Op::BLOCK) op.load_state(state, q, u0, w.ch);
    };
    if (lo < hi) load_tile(std::true_type{}, lo);
    float CA[V], c[V];                                                  // AGG: (CA, c) is the composition so far; else c is the state
    if (AGG) {
#pragma unroll
        for (int v = 0; v < V; ++v) { CA[v] = 1.f; c[v] = 0.f; }
    } else {
        op.carry0(c, w.ch);
        if (split > 0) {                                                // the stretches before this one, a part of them by each wave
            float PA[V], PS[V];
#pragma unroll
            for (int v = 0; v < V; ++v) { PA[v] = 1.f; PS[v] = 0.f; }
            const int j1 = (wave + 1) * split / NW;
            int j = wave * split / NW;
            auto join = [&](const float (&m)[2 * V]) __attribute__((always_inline)) {
#pragma unroll
                for (int v = 0; v < V; ++v) { PS[v] = through<CUTS>(m[2 * v], m[2 * v + 1], PS[v]); PA[v] = joined<CUTS>(m[2 * v], PA[v]); }
            };
            for (; j + 16 <= j1; j += 16) {                             // (sixteen loads in flight: another XCD wrote them, they come from memory)
                float m[16][2 * V];
#pragma unroll
                for (int k = 0; k < 16; ++k) load_vec<float, 2 * V>(m[k], q.ws, ((int64_t)(j + k) * q.C + w.ch) * 2);
#pragma unroll
                for (int k = 0; k < 16; ++k) join(m[k]);
            }
            float m[16][2 * V];
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (j + k < j1) load_vec<float, 2 * V>(m[k], q.ws, ((int64_t)(j + k) * q.C + w.ch) * 2);
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (j + k < j1) join(m[k]);
#pragma unroll
            for (int v = 0; v < V; ++v) { ex[0][wave][0][lane][v] = PA[v]; ex[0][wave][1][lane][v] = PS[v]; }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < NW; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) c[v] = through<CUTS>(ex[0][k][0][lane][v], ex[0][k][1][lane][v], c[v]);
        }
    }
    SpreadSum sum;                                                      // (moments: of this thread's values)
    int par = 1;                                                        // (the half the stretches were not left in)
    // FULL: every step of the tile lies inside the stretch.  NEXT: the next tile is 0 none, 1 perhaps partly beyond the end, 2 full.
    auto work = [&](auto full, auto next, int tile) __attribute__((always_inline)) {
        constexpr bool FULL = decltype(full)::value;
        constexpr int NEXT = decltype(next)::value;
        const int u0 = tile + wave * L;
        typename Op::Item it[L];
        float PA[V], PS[V], mine[V];                                    // mine: the state in front of this wave's steps
        bool any[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { PA[v] = 1.f; PS[v] = 0.f; any[v] = false; mine[v] = c[v]; }
        if constexpr (Op::BLOCK) op.states(it, raw, state, ln, q.T - 1 - u0, FULL ? L : hi - u0);
#pragma unroll
        for (int l = 0; l < L; ++l) {
            op.coef(it[l], raw[l], ln, step_at(u0, l), FULL || u0 + l < hi);
            if (NW > 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const bool cut = CUTS && cut_of(it[l], v);
                    PS[v] = __fmaf_rn(it[l].A[v], cut ? 0.f : PS[v], it[l].S[v]);
                    PA[v] *= it[l].A[v];
                    any[v] = any[v] || cut;
                }
            }
        }
        if constexpr (NEXT != 0) load_tile(std::bool_constant<NEXT == 1>{}, tile + NW * L);
        if constexpr (NW > 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) { ex[par][wave][0][lane][v] = CUTS && any[v] ? -0.f : PA[v]; ex[par][wave][1][lane][v] = PS[v]; }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                if (k == wave) {
#pragma unroll
                    for (int v = 0; v < V; ++v) mine[v] = c[v];
                }
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float A = ex[par][k][0][lane][v], S = ex[par][k][1][lane][v];
                    c[v] = through<CUTS>(A, S, c[v]);
                    if (AGG) CA[v] = joined<CUTS>(A, CA[v]);
                }
            }
            par ^= 1;                                                   // (the next tile's pairs go to the other half: one barrier a tile)
        }
        if (!AGG) {
            const int kept = (q.T - u0) & 7;                            // the step of these, if any, in front of which the state is kept
            float front[V];
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const bool on = have && (FULL || u0 + l < hi);
                if constexpr (Op::KEEPS) {
#pragma unroll
                    for (int v = 0; v < V; ++v) front[v] = l == 0 || l == kept ? mine[v] : front[v];
                }
                if constexpr (Op::SUMS) op.step(mine, it[l], ln, step_at(u0, l), on, sum);
                else op.step(mine, it[l], ln, step_at(u0, l), on);
            }
            if constexpr (Op::KEEPS) {
                if (op.ck && have && kept < L && u0 + kept < hi) store_vec<float, V>(op.ck, (int64_t)((q.T - u0) / 8 - 1) * q.C + w.ch, front);
            }
            if (NW == 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) c[v] = mine[v];
            }
        }
    };
    int tile = lo;
    for (; tile + 2 * NW * L <= hi; tile += NW * L) work(std::true_type{}, std::integral_constant<int, 2>{}, tile);
    if (tile + NW * L < hi) { work(std::true_type{}, std::integral_constant<int, 1>{}, tile); tile += NW * L; }
    if (tile < hi) work(std::false_type{}, std::integral_constant<int, 0>{}, tile);
    if (AGG) {
        if (have && wave == 0) {
            float m[2 * V];
#pragma unroll
            for (int v = 0; v < V; ++v) { m[2 * v] = CA[v]; m[2 * v + 1] = c[v]; }
            store_vec<float, 2 * V>(q.ws, ((int64_t)split * q.C + w.ch) * 2, m);
        }
        return;
    }
    if (have && wave == 0 && split == q.nsplit - 1) op.finish(c, w.ch);
    if constexpr (Op::MOMENTS) {
        __shared__ double red[NW][3];
        const Spread ws = wave_join(sum.spread());
        if (lane == 0) { red[wave][0] = ws.n; red[wave][1] = ws.mean; red[wave][2] = ws.m2; }
        __syncthreads();
        if (threadIdx.x == 0) {
            Spread t = ws;
            for (int k = 1; k < NW; ++k) t = join(t, {red[k][0], red[k][1], red[k][2]});
            double *to = mom + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 3;
            to[0] = t.n; to[1] = t.mean; to[2] = t.m2;
        }
    }
}

// The backward pass of many channels, one wave for all of time, from the states that the forward pass kept: it reads gate, x, dh
// and an eighth of a state instead of gate, x, dh and h (200 x 1920 x 256 float32: 386 us for 2.0 GB, 460 us with h).
template <typename T, int V, bool MSK>
__global__ __launch_bounds__(64) void k_scan_back_kept(BackwardKeptOp<T, V, MSK, uint32_t> op, ScanGeom q)
{
    constexpr int L = 8;
    typedef BackwardKeptOp<T, V, MSK, uint32_t> Op;
    const uint32_t first = blockIdx.x * 64u * V, mine_ch = first + threadIdx.x * V;
    const bool have = mine_ch < q.C;
    Place w;
    w.ch = have ? mine_ch : first;
    w.b0 = __builtin_amdgcn_readfirstlane(first / q.D);
    const uint32_t rel = w.ch - w.b0 * q.D;
    w.db = rel / q.D;
    w.d = rel - w.db * q.D;
    const typename Op::Lane ln = op.lane(q, w);
    struct Raw { Words<T, V> g, x, dh; Words<uint8_t, 1> cut; };
    Raw raw[L];
    float state[V], c[V];
    // the block of steps t0 .. t0 + 7; CLAMP: one that begins in front of the first step reads that one again
    auto load = [&](auto clamp, int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const Step s = decltype(clamp)::value ? Step{t0 + l > 0 ? t0 + l : 0, 0} : Step{t0, l};
            fetch(raw[l].g, ln.g, step_off(s, op.gate.st), ln.og);
            fetch(raw[l].x, ln.x, step_off(s, op.x.st), ln.ox);
            if (op.dh.p) fetch(raw[l].dh, ln.dh, step_off(s, op.dh.st), ln.odh);
            if (MSK) { raw[l].cut.w = 0; if (op.marks.resets) fetch(raw[l].cut, ln.r, step_off(s, op.marks.r_st), ln.m.r); }
        }
        op.load_state(state, q, q.T - L - t0, w.ch);
    };
    op.carry0(c, w.ch);
    // FULL: all eight steps are there.  NEXT: the block in front of this one is 0 none, 1 perhaps not full, 2 full
    auto work = [&](auto full, auto next, int t0) __attribute__((always_inline)) {
        constexpr bool FULL = decltype(full)::value;
        constexpr int NEXT = decltype(next)::value;
        float a[L][V], b[L][V], m[L][V], dh[L][V], h[V];
        bool cut[L];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = state[v];
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const bool on = (FULL || t0 + l >= 0) && (!MSK || t0 + l < ln.m.len);
            cut[l] = MSK && raw[l].cut.get(0);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gate_pair(raw[l].g.get(v), a[l][v], b[l][v]);
                const float before = cut[l] ? 0.f : h[v], x = raw[l].x.get(v);
                m[l][v] = (before - x) * a[l][v];
                dh[l][v] = op.dh.p ? raw[l].dh.get(v) : 0.f;
                const float after = __fmaf_rn(a[l][v], before, b[l][v] * x);
                h[v] = on ? after : h[v];
            }
        }
        if constexpr (NEXT != 0) load(std::bool_constant<NEXT == 1>{}, t0 - L);
#pragma unroll
        for (int l = L - 1; l >= 0; --l) {
            const bool in = FULL || t0 + l >= 0, on = in && (!MSK || t0 + l < ln.m.len);
            float og[V], ox[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float G = dh[l][v] + c[v], gx = G * b[l][v];
                ox[v] = on ? gx : 0.f;
                og[v] = on ? gx * m[l][v] : 0.f;
                c[v] = on ? (cut[l] ? 0.f : a[l][v] * G) : c[v];
            }
            if (have && in) {
                put<T, V>(ln.dg, step_off(Step{t0, l}, op.dgate.st), ln.odg, og);
                put<T, V>(ln.dx, step_off(Step{t0, l}, op.dx.st), ln.odx, ox);
            }
        }
    };
    int t0 = q.T - L;
    load(std::true_type{}, t0);
    for (; t0 >= L; t0 -= L) work(std::true_type{}, std::integral_constant<int, 2>{}, t0);
    if (t0 > 0) { work(std::true_type{}, std::integral_constant<int, 1>{}, t0); t0 -= L; }
    work(std::false_type{}, std::integral_constant<int, 0>{}, t0);
    if (have) op.finish(c, w.ch);
}

// (480 partials: 4.7 us, a launch and three trips to memory.)
// One workgroup: (mean, 1 / (standard deviation + 1e-8)) of the advantages from the partials of k_scan.
__global__ __launch_bounds__(256) void k_moments(const double *mom, int64_t n, float *out)
{
    __shared__ double red[4][3];
    Spread s{0, 0, 0};
    for (int64_t k = threadIdx.x; k < n; k += 256) s = join(s, {mom[k * 3], mom[k * 3 + 1], mom[k * 3 + 2]});
    s = wave_join(s);
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6][0] = s.n; red[threadIdx.x >> 6][1] = s.mean; red[threadIdx.x >> 6][2] = s.m2; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 4; ++k) s = join(s, {red[k][0], red[k][1], red[k][2]});
        out[0] = (float)s.mean;
        out[1] = (float)(1.0 / (sqrt(s.n > 0.0 ? s.m2 / s.n : 0.0) + 1e-8));
    }
}

// (122880 x 256 float32: 113 us for 630 MB, bound by HBM; 30 x 64: 2.2 us, a launch.)
// One step of the memory: state <- a k state + (1 - a) x, out = the new state in the inputs' type.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_scan_step(uint32_t n, uint32_t D, const void *gate, int64_t g_sb, const void *x, int64_t x_sb,
                                                   float *state, const uint8_t *reset, int64_t r_sb, void *out, int64_t o_sb)
{
    const uint32_t e = (blockIdx.x * 256 + threadIdx.x) * V;
    if (e >= n) return;
    const int64_t b = e / D, d = e - (uint32_t)b * D;
    float g[V], xv[V], s[V];
    load_vec<T, V>(g, gate, b * g_sb + d);
    load_vec<T, V>(xv, x, b * x_sb + d);
    load_vec<float, V>(s, state, e);
    const bool cut = reset && reset[b * r_sb];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float a, k;
        gate_pair(g[v], a, k);
        s[v] = __fmaf_rn(cut ? 0.f : a, cut ? 0.f : s[v], k * xv[v]);
    }
    store_vec<float, V>(state, e, s);
    store_vec<T, V>(out, b * o_sb + d, s);
}
