// What the row operators (token scores, top-entry distillation) share: how a row of logits of any size and alignment is
// cut into 16-byte vectors, the softmax statistics of a row, and the selection of its largest entries. Internal.
#pragma once
#include "cwrnnt_common.cuh"

namespace cwrnnt {

constexpr int kRowThreads = 256;  // threads of a CTA in the row operators
constexpr int kFewRowLanes = 512; // lanes of a long row where there are fewer rows than SMs

// ------------------------------------------------------------------------------------------------ rows as vectors
// A row is read in 16-byte vectors that lie on 16-byte boundaries, whatever V and the row stride. What lies before the
// first boundary and behind the last is put together element by element, with -inf outside the row, so nothing outside
// it is read. What a launch knows of its rows:
//   kAny      nothing
//   kAligned  every row starts and ends on a 16-byte boundary
//   kFull     the same, and a row is exactly the vectors that its lanes hold in registers
enum { kAny = 0, kAligned = 1, kFull = 2 };

// The edges, out of line: they would fill the instruction cache from within every unrolled loop.
template <typename T>
__device__ __noinline__ uint4 load_edge(const T *row, int first, int V)
{
    using E = Elt<T>;
    typename E::acc e[E::VE];
#pragma unroll
    for (int c = 0; c < E::VE; ++c) {
        const int k = first + c;
        e[c] = k >= 0 && k < V ? E::to_acc(__ldg(row + k)) : typename E::acc(-INFINITY);
    }
    return E::pack(e);
}
template <typename T>
__device__ __noinline__ void store_edge(T *out, int first, int V, uint4 v)
{
    const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
    for (int c = 0; c < Elt<T>::VE; ++c)
        if (first + c >= 0 && first + c < V) out[first + c] = e[c];
}

template <typename T>
__device__ __forceinline__ uint4 vector_of_nothing()
{
    if constexpr (sizeof(T) == 2) {
        const uint32_t w = Elt<T>::kBf16 ? 0xff80ff80u : 0xfc00fc00u;
        return make_uint4(w, w, w, w);
    } else if constexpr (sizeof(T) == 4) {
        return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
    } else {
        return make_uint4(0u, 0xfff00000u, 0u, 0xfff00000u);
    }
}

// The whole vectors come first (0 .. whole_count-1, one load each), then the edges, if there are any: the elements before
// the first boundary, then those behind the last.
template <typename T, int MODE>
struct RowVectors {
    static constexpr int VE = Elt<T>::VE;
    const T *row;
    int V, lead, whole_count, count;  // lead: elements before the first boundary
    __device__ __forceinline__ RowVectors(const T *row_, int V_) : row(row_), V(V_)
    {
        if (MODE != kAny) {
            lead = 0;
            count = whole_count = V_ / VE;
            return;
        }
        lead = int((16 - (reinterpret_cast<uintptr_t>(row_) & 15)) & 15) / int(sizeof(T));
        if (lead > V_) {  // the row lies between two boundaries
            whole_count = 0;
            count = 1;
        } else {
            whole_count = (V_ - lead) / VE;
            count = whole_count + (lead > 0) + (lead + whole_count * VE < V_);
        }
    }
    __device__ __forceinline__ bool whole(int i) const { return MODE != kAny || i < whole_count; }
    // first element of vector i (before the row, if it is the leading edge)
    __device__ __forceinline__ int first(int i) const
    {
        if (MODE != kAny) return i * VE;
        return i < whole_count ? lead + i * VE : (i == whole_count && lead > 0 ? lead - VE : lead + whole_count * VE);
    }
    // where element k lies: vector * VE + place in it
    __device__ __forceinline__ int place(int k) const
    {
        if (MODE != kAny) return k;
        const int behind = lead + whole_count * VE;
        if (k < lead) return whole_count * VE + k - (lead - VE);
        if (k >= behind) return (whole_count + (lead > 0)) * VE + k - behind;
        return k - lead;
    }
    __device__ __forceinline__ uint4 load(int i) const
    {
        if (whole(i)) return __ldg(reinterpret_cast<const uint4 *>(row + lead) + i);
        return load_edge(row, first(i), V);
    }
    // vectors lane, lane + LANES, .. of the row into registers
    template <int LANES, int NV>
    __device__ __forceinline__ void load_all(uint4 (&v)[NV], int lane, bool active) const
    {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            v[j] = vector_of_nothing<T>();
            if (MODE == kFull ? active : active && j * LANES + lane < count) v[j] = load(j * LANES + lane);
        }
    }
    // f(i, v) for all vectors of the row, four a lane at a time (v[j] is vector i + j * LANES, nothing behind the last):
    // straight loads but for the last of them
    template <int LANES, typename F>
    __device__ __forceinline__ void sweep(int lane, bool seen, F &&f) const
    {
#pragma unroll 1
        for (int at = 0; at < count; at += 4 * LANES) {
            uint4 v[4];
            if (seen && at + 4 * LANES <= whole_count) {
                const uint4 *p = reinterpret_cast<const uint4 *>(row + lead) + at + lane;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = __ldg(p + j * LANES);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = vector_of_nothing<T>();
                    if (seen && at + j * LANES + lane < count) v[j] = load(at + j * LANES + lane);
                }
            }
            f(at + lane, v);
        }
    }
    // Stores vector i of a row of gradients. `same`: the output row has the input row's alignment, so that vector i is
    // one 16-byte store; else element by element.
    template <bool FIRST_OUT = false>
    __device__ __forceinline__ void store(T *out, int i, bool same, const typename Elt<T>::acc (&e)[VE]) const
    {
        const uint4 v = Elt<T>::pack(e);
        uint4 *const to = reinterpret_cast<uint4 *>(out + lead) + i;
        if (MODE != kAny || (same && whole(i))) {
            if (FIRST_OUT)
                st_stream(to, v);
            else
                *to = v;
        } else {
            store_edge(out, first(i), V, v);
        }
    }
};

// ---------------------------------------------------------------------------------------------- softmax of a row
// With temperature tau and kappa = log2(e)/tau, a term of the row's softmax is 2^(x*kappa - shift): one FFMA and one
// ex2 in float (relative error near 2^-22). The shift is the row's (or thread's) maximum in these units, rounded to
// float once; where the sum's logarithm is taken, that rounding is undone. Beyond 2^24 (2^53 in double) the rounding moves
// the shift by whole units: a row masked with -1e10 would be off by 2^440 before it is undone. There a term is formed from
// the difference, 2^((x - max) * kappa), which has no shift to round. Double takes exp2 and log2 of the library.
template <typename A>
struct Base2;
template <>
struct Base2<float> {
    static __device__ __forceinline__ float exp2_of(float d) { return ex2_approx(d); }
    static __device__ __forceinline__ float ln_of(float s) { return logf(s); }
    static __device__ __forceinline__ float fma_of(float a, float b, float c) { return fmaf(a, b, c); }
    static __device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
    static __device__ __forceinline__ float ratio(float a, float b) { return __fdividef(a, b); }  // b in [2^-126, 2^126]
    // below this exponent a term is zero; it keeps 0 * (-inf) out of sum p log p
    static constexpr float kFloor = -1000.0f;
    // largest shift that x*kappa - shift is formed with: its rounding is below one there, a factor of two at most
    static constexpr float kMostShift = 16777216.0f;
};
template <>
struct Base2<double> {
    static __device__ __forceinline__ double exp2_of(double d) { return exp2(d); }
    static __device__ __forceinline__ double ln_of(double s) { return log(s); }
    static __device__ __forceinline__ double fma_of(double a, double b, double c) { return fma(a, b, c); }
    static __device__ __forceinline__ double max_of(double a, double b) { return fmax(a, b); }
    static __device__ __forceinline__ double ratio(double a, double b) { return a / b; }
    static constexpr double kFloor = -5000.0;
    static constexpr double kMostShift = 9007199254740992.0;
};

constexpr double kLn2 = 0.6931471805599453;
constexpr double kLog2e = 1.4426950408889634;

// Running statistics of (part of) a row: maximum x, s = sum 2^d and t = sum 2^d d with d = (x - max) * kappa.
template <typename A>
struct RowStats {
    A max, s, t;
    __device__ __forceinline__ void clear()
    {
        max = A(-INFINITY);
        s = t = A(0);
    }
    static __device__ __forceinline__ A shift_of(A max, A kappa)
    {
        return max == A(-INFINITY) ? A(0) : max * kappa;
    }
    // (true for a maximum of +inf as well: its terms are then inf - inf = NaN, as they must be)
    static __device__ __forceinline__ bool extreme(A shift) { return !(fabs(shift) <= Base2<A>::kMostShift); }
    // Brings the sums to a maximum that is at least the present one.
    template <bool ENT>
    __device__ __forceinline__ void raise(A new_max, A kappa)
    {
        using M = Base2<A>;
        const A from = shift_of(max, kappa), to = shift_of(new_max, kappa);
        A by = from - to;  // <= 0, or NaN
        // sums formed from differences know no shift: theirs is the maximum itself
        if (extreme(from) || extreme(to)) by = (max - new_max) * kappa - excess_of(max, kappa) + excess_of(new_max, kappa);
        // nothing summed yet: the sums stay zero whatever the difference is
        const A f = s == A(0) ? A(1) : M::exp2_of(by);
        if (ENT && s != A(0)) t = f == A(0) ? A(0) : (t + s * by) * f;
        s *= f;
        max = new_max;
    }
    template <bool ENT>
    __device__ __forceinline__ void join(const RowStats &o, A kappa)
    {
        RowStats b = o;
        const A m = Base2<A>::max_of(max, b.max);
        raise<ENT>(m, kappa);
        b.raise<ENT>(m, kappa);
        s += b.s;
        if (ENT) t += b.t;
    }
    // no finite entry (and no NaN either)
    __device__ __forceinline__ bool nothing() const { return max == A(-INFINITY) && s == s; }
    // log2 of the factor by which the rounding of the shift has made the sums too large
    static __device__ __forceinline__ A excess_of(A max, A kappa)
    {
        const A shift = shift_of(max, kappa);
        if (extreme(shift) || max == A(-INFINITY)) return A(0);
        return Base2<A>::fma_of(max, kappa, -shift);
    }
    __device__ __forceinline__ A excess(A kappa) const { return excess_of(max, kappa); }
    // sum 2^((x - max) * kappa)
    __device__ __forceinline__ A sum(A kappa) const { return s * Base2<A>::exp2_of(-excess(kappa)); }
};

// What a row's log-probabilities are taken from, and its entropy ln s - ln2 * t / s: of a row's joined statistics.
template <typename A>
struct RowLog {
    A max, sum, ln_s, entropy;
    __device__ __forceinline__ RowLog(const RowStats<A> &st, A kappa) : max(st.max)
    {
        using M = Base2<A>;
        const A over = st.excess(kappa), ln = M::ln_of(st.s);
        sum = st.s * M::exp2_of(-over);
        ln_s = st.nothing() ? A(0) : ln - A(kLn2) * over;
        entropy = st.s == A(0) ? A(0) : ln - A(kLn2) * M::ratio(st.t, st.s);
    }
};

// ln of an entry's probability, (x - max) / tau - ln s: log-probabilities near zero keep their digits, and so do those
// of rows of the type's lowest value.
template <typename A>
__device__ __forceinline__ A log_prob_of(A x, A max, A inv_tau, A ln_s)
{
    return x == A(-INFINITY) ? (ln_s == ln_s ? A(-INFINITY) : A(NAN)) : Base2<A>::fma_of(x - max, inv_tau, -ln_s);
}

// The statistics of a row over the lanes of a warp that hold its parts: to the common maximum, then added up.
template <int LANES, bool ENT, typename A>
__device__ __forceinline__ void join_lanes(RowStats<A> &st, A kappa)
{
    A m = st.max;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = Base2<A>::max_of(m, __shfl_xor_sync(0xffffffffu, m, o));
    st.template raise<ENT>(m, kappa);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
        if (ENT) st.t += __shfl_xor_sync(0xffffffffu, st.t, o);
    }
}

// The same over the warps of a CTA, whose joined statistics lie in `parts`: added up in the warps' order, the same bits in
// every thread.
template <int WARPS, bool ENT, typename A>
__device__ __forceinline__ RowStats<A> join_warps(const RowStats<A> *parts, A kappa)
{
    RowStats<A> st;
    st.clear();
    A m = parts[0].max;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) m = Base2<A>::max_of(m, parts[w].max);
#pragma unroll 1
    for (int w = 0; w < WARPS; ++w) {
        RowStats<A> part = parts[w];
        part.template raise<ENT>(m, kappa);
        st.s += part.s;
        if (ENT) st.t += part.t;
    }
    st.max = m;
    return st;
}

// How a row's (or a thread's) terms are formed at a fixed maximum: as x*kappa - shift, or from the difference to the
// maximum where the shift's rounding would count (rows of a mask's value, up to the type's lowest). `floored`: a floor under x is far below any term
// that counts, so it may keep 0 * (-inf) out of sum p log p.
template <typename T>
struct TermsAt {
    using A = typename Elt<T>::acc;
    A max, shift;
    bool plain, floored;
    __device__ __forceinline__ TermsAt(A max_, A kappa)
        : max(max_ == A(-INFINITY) ? A(0) : max_), shift(RowStats<A>::shift_of(max_, kappa))
    {
        plain = !RowStats<A>::extreme(shift);
        floored = sizeof(T) == 2 && plain && (Elt<T>::floor() - max) * kappa < A(-200);
    }
    __device__ __forceinline__ A exponent(A x, A kappa) const
    {
        return plain ? Base2<A>::fma_of(x, kappa, -shift) : (x - max) * kappa;
    }
};

// Adds one vector's terms to s = sum 2^d and, ENT, t = sum 2^d d.
template <typename T, bool ENT>
__device__ __forceinline__ void add_terms(uint4 v, typename Elt<T>::acc kappa, const TermsAt<T> &at,
                                          typename Elt<T>::acc &s, typename Elt<T>::acc &t)
{
    using E = Elt<T>;
    using A = typename E::acc;
    using M = Base2<A>;
    constexpr bool kFloors = ENT && sizeof(T) == 2;
    A e[E::VE];
    if (kFloors ? at.floored : at.plain) {
        if constexpr (kFloors) v = E::at_least_floor(v);
        E::unpack(v, e);
#pragma unroll
        for (int c = 0; c < E::VE; ++c) {
            const A d = M::fma_of(e[c], kappa, -at.shift), w = M::exp2_of(d);
            s += w;
            if (ENT) t = M::fma_of(w, kFloors ? d : M::max_of(d, M::kFloor), t);
        }
    } else {
        E::unpack(v, e);
#pragma unroll
        for (int c = 0; c < E::VE; ++c) {
            const A d = at.exponent(e[c], kappa), w = M::exp2_of(d);
            s += w;
            if (ENT) t = M::fma_of(w, M::max_of(d, M::kFloor), t);
        }
    }
}

// ------------------------------------------------------------------------------------------- largest entries
// A total order of a row's entries in which "first" is the larger value and, among equal values, the lower index; NaN
// comes before everything, -0 equals +0. Floats and 16-bit types pack value and index into one 64-bit word.
template <typename A>
struct TopKey;
template <>
struct TopKey<float> {
    uint64_t k;
    static __device__ __forceinline__ TopKey of(float v, int index)
    {
        v += 0.0f;  // -0 -> +0
        const uint32_t b = __float_as_uint(v);
        const uint32_t o = v != v ? 0xfffffffeu : (b & 0x80000000u ? ~b : b | 0x80000000u);
        return TopKey{(uint64_t(o) << 32) | uint32_t(~uint32_t(index))};
    }
    static __device__ __forceinline__ TopKey none() { return TopKey{0}; }            // after every entry
    static __device__ __forceinline__ TopKey all() { return TopKey{~uint64_t(0)}; }  // before every entry
    __device__ __forceinline__ bool before(const TopKey &o) const { return k > o.k; }
    __device__ __forceinline__ int index() const { return int(~uint32_t(k)); }
};
template <>
struct TopKey<double> {
    uint64_t o;
    uint32_t i;  // complement of the index
    static __device__ __forceinline__ TopKey of(double v, int index)
    {
        v += 0.0;
        const uint64_t b = uint64_t(__double_as_longlong(v));
        const uint64_t ord = v != v ? ~uint64_t(1) : (b >> 63 ? ~b : b | (uint64_t(1) << 63));
        return TopKey{ord, ~uint32_t(index)};
    }
    static __device__ __forceinline__ TopKey none() { return TopKey{0, 0}; }
    static __device__ __forceinline__ TopKey all() { return TopKey{~uint64_t(0), ~uint32_t(0)}; }
    __device__ __forceinline__ bool before(const TopKey &x) const { return o > x.o || (o == x.o && i > x.i); }
    __device__ __forceinline__ int index() const { return int(~i); }
};
__device__ __forceinline__ TopKey<float> shfl_xor_key(unsigned mask, const TopKey<float> &k, int by)
{
    return TopKey<float>{__shfl_xor_sync(mask, k.k, by)};
}
__device__ __forceinline__ TopKey<double> shfl_xor_key(unsigned mask, const TopKey<double> &k, int by)
{
    return TopKey<double>{__shfl_xor_sync(mask, k.o, by), __shfl_xor_sync(mask, k.i, by)};
}

// The same order in 32 bits for the 16-bit types' rows of at most 65 535 entries; 0 comes after every entry.
template <typename T>
__device__ __forceinline__ uint32_t short_key(T v, int index)
{
    const float f = Elt<T>::to_acc(v) + 0.0f;  // -0 -> +0
    const uint32_t b = __float_as_uint(f);
    uint32_t o;
    if constexpr (Elt<T>::kBf16) {
        o = b >> 16;
    } else {
        o = uint32_t(__half_as_ushort(__float2half_rn(f)));
    }
    o = o & 0x8000u ? ~o & 0xffffu : o | 0x8000u;
    return (o << 16) | (0xffffu - uint32_t(index));
}

// Which elements of a vector are at least `bar` (no NaN among them): bit c for element c.
template <typename T>
__device__ __forceinline__ uint32_t at_least(const uint4 &v, typename Elt<T>::acc bar)
{
    using E = Elt<T>;
    uint32_t bits = 0;
    if constexpr (sizeof(T) == 2) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        using T2 = typename E::pair;
        const T2 b2 = E::both(bar);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t m = __hge2_mask(*reinterpret_cast<const T2 *>(&w[i]), b2);
            bits |= m & ((1u << (2 * i)) | (1u << (2 * i + 1 + 16)));
        }
        bits = (bits | (bits >> 16)) & 0xffu;
    } else {
        typename E::acc e[E::VE];
        E::unpack(v, e);
#pragma unroll
        for (int c = 0; c < E::VE; ++c) bits |= e[c] >= bar ? 1u << c : 0u;
    }
    return bits;
}

// The same for vector i of a row, without the elements before and behind the row.
template <typename T, int MODE>
__device__ __forceinline__ uint32_t at_least(const RowVectors<T, MODE> &rv, int i, const uint4 &v,
                                             typename Elt<T>::acc bar)
{
    uint32_t hit = at_least<T>(v, bar);
    if (MODE == kAny && !rv.whole(i)) {
        const int f = rv.first(i);
        if (f < 0) hit &= ~0u << (-f);
        if (rv.V - f < Elt<T>::VE) hit &= rv.V > f ? (1u << (rv.V - f)) - 1u : 0u;
    }
    return hit;
}

// The best key of vector `i` of a row that comes after `last` in the order.
template <typename T, int MODE>
__device__ __forceinline__ void best_after(const RowVectors<T, MODE> &rv, int i, const uint4 &v,
                                           const TopKey<typename Elt<T>::acc> &last,
                                           TopKey<typename Elt<T>::acc> &best)
{
    using E = Elt<T>;
    using Key = TopKey<typename E::acc>;
    typename E::acc e[E::VE];
    E::unpack(v, e);
#pragma unroll
    for (int c = 0; c < E::VE; ++c) {
        const int k = rv.first(i) + c;
        if (MODE == kAny && (k < 0 || k >= rv.V)) continue;
        const Key key = Key::of(e[c], k);
        if (last.before(key) && key.before(best)) best = key;
    }
}

}  // namespace cwrnnt
