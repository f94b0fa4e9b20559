// Distillation of logits rows from a teacher's top entries, loss and gradient in one pass. Row r has K entries: a token
// c_i and the teacher's value a_i for it. With p = softmax(x / tau) of the student's row:
//   with a tail      a_i are the teacher's log-probabilities: q_i = exp a_i, q_rest = 1 - sum q_i, and every token that
//                    is not listed belongs to one class of its own, p_rest = sum of their p_j:
//                        D = sum_i q_i (a_i - ln p_{c_i}) + q_rest (ln q_rest - ln p_rest)
//   without          a_i are logits or log-probabilities, renormalised over the list: q = softmax(a / tau),
//                        D = sum_i q_i (ln q_i - ln p_{c_i})
//   gradient         dD/dx_j = (1/tau) ( Q p_j - sum of the q_i with c_i = j )          listed, Q = all of q
//                            = (1/tau) ( Q p_rest - q_rest ) p_j / p_rest              not listed, with a tail
//                            = (1/tau) Q p_j                                           not listed, without
// The rest class is summed by itself, with its own maximum (listed entries are blanked before the sums): as one minus
// the listed probabilities it would lose all its digits where the student is sure of a listed token, and its gradient
// divides nothing by a small number.
//
// Bound: HBM, 2 * V * sizeof(element) bytes a row: rows of up to 512 vectors (8 KB) stay in registers between the sums
// and the gradient; longer ones take a CTA each, whose second reading comes from L2.
// The summed loss is added up in a fixed order: rows in their CTA, then the CTAs' sums in a second small kernel.
#include "cwrnnt_kernels.h"
#include "cwrnnt_rowops.cuh"

namespace cwrnnt {

namespace {

template <typename T>
struct DistillArgs {
    using A = typename Elt<T>::acc;
    using C = typename Elt<T>::cost;
    const T *x;
    T *gx;  // null: loss only
    int64_t n_rows, x_stride, g_stride;
    int V, K, KP;  // KP: K up to a power of two
    A kappa;       // log2(e) / tau
    A inv_tau;     // 1 / tau
    double scale;  // of the summed loss and of the gradient
    const C *teacher, *weight, *upstream;
    int upstream_stride;
    const int32_t *index;
    C *row_loss;
    double *partial;  // one sum per CTA
};

// e^a to 2^-33 relative, for a <= 0 and a little above, in a dozen double operations: 2^n times the series of e^r,
// |r| <= ln2 / 2 (its first omitted term: 0.347^9 / 9! = 2e-10). What the teacher leaves for the rest is one minus a sum
// of these, and a float's digits would not do for that.
__device__ __forceinline__ double exp_mid(double a)
{
    if (!(a > -700.0)) return a != a ? a : 0.0;
    if (a > 700.0) return INFINITY;
    const double n = rint(a * kLog2e), r = fma(n, -kLn2, a);
    double p = 1.0 / 40320.0;
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return p * __hiloint2double((int(n) + 1023) << 20, 0);
}
__device__ __forceinline__ double teacher_exp(double a, float) { return exp_mid(a); }
__device__ __forceinline__ double teacher_exp(double a, double) { return exp(a); }

// Sums and maxima over the lanes of a row that hold its entries: lanes 0 .. KP-1 (a power of two, the others hold the
// neutral element), the result in every lane of the row. All lanes of a warp call these together.
template <int LPR, typename V>
__device__ __forceinline__ V entry_sum(V v, int KP)
{
    for (int o = KP >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return __shfl_sync(0xffffffffu, v, 0, LPR);
}
template <int LPR, typename V>
__device__ __forceinline__ V entry_max(V v, int KP)
{
    for (int o = KP >> 1; o > 0; o >>= 1) v = Base2<V>::max_of(v, __shfl_xor_sync(0xffffffffu, v, o));
    return __shfl_sync(0xffffffffu, v, 0, LPR);
}

// One row's teacher entry, held by lane e of the row's lanes, and what follows from all of them.
template <typename A>
struct Entries {
    int c;       // token, -1: none
    bool first;  // no earlier entry names the same token
    bool bad;    // some token of the row lies outside it
    A q, lq;     // teacher's probability and its logarithm
    A sum_q;     // over the row
    A left;      // one minus that, at least 0
    A dup_q;     // q of all entries with this token, added up in their order
};

// All lanes of a warp call this together; LPR lanes belong to a row, lane `gl` of them holds entry gl: token `c`, value
// `a` (-1, -inf: none).
template <int LPR, bool TAIL, typename A>
__device__ __forceinline__ Entries<A> weigh_entries(int c, A a, int V, int K, int KP, A inv_tau, int gl)
{
    constexpr unsigned kAll = 0xffffffffu;
    using M = Base2<A>;
    Entries<A> en;
    const unsigned outside = __ballot_sync(kAll, c >= V);
    en.bad = ((outside >> ((threadIdx.x & 31) / LPR * LPR)) & (LPR == 32 ? kAll : (1u << (LPR & 31)) - 1u)) != 0;
    en.c = c < 0 || c >= V ? -1 : c;
    if (en.c < 0) a = A(-INFINITY);
    if (TAIL) {
        en.lq = a;
        const double q = teacher_exp(double(a), A(0));
        const double sum = entry_sum<LPR>(q, KP);
        en.q = A(q);
        en.sum_q = A(sum);
        en.left = A(fmax(0.0, 1.0 - sum));
    } else {
        const A z = a * inv_tau;
        const A m = entry_max<LPR>(z, KP);
        const A w = m == A(-INFINITY) ? A(0) : M::exp2_of((z - m) * A(kLog2e));
        const A s = entry_sum<LPR>(w, KP);
        en.lq = s == A(0) ? A(-INFINITY) : z - m - M::ln_of(s);
        en.q = s == A(0) ? A(0) : M::ratio(w, s);
        en.sum_q = s == A(0) ? A(0) : s / s;
        en.left = A(0);
    }
    en.first = en.c >= 0;
    en.dup_q = A(0);
    for (int o = 0; o < K; ++o) {
        const int other = __shfl_sync(kAll, en.c, o, LPR);
        const A oq = __shfl_sync(kAll, en.q, o, LPR);
        const bool mine = other == en.c;
        en.dup_q += mine ? oq : A(0);
        en.first = en.first && !(mine && o < gl);
    }
    return en;
}

// Element c of a vector becomes -inf.
template <typename T>
__device__ __forceinline__ void blank_element(uint4 &v, int c)
{
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (sizeof(T) == 2) {
        const uint32_t ninf = Elt<T>::kBf16 ? 0xff80ff80u : 0xfc00fc00u, mask = c & 1 ? 0xffff0000u : 0x0000ffffu;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k == c >> 1) w[k] = (w[k] & ~mask) | (ninf & mask);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k == c) w[k] = 0xff800000u;
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (k == c) w[2 * k] = 0u, w[2 * k + 1] = 0xfff00000u;
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
}

// What the row's statistics and entries give: its divergence, and its gradient's factors. The gradient is
//     2^((x - top) * kappa) * factor                                   where no entry names the token
//     2^((x - all_top) * kappa) * all_factor - q_factor * dup_q        where one does
template <typename A>
struct RowResult {
    A loss;  // weighted
    A top, factor;
    A all_top, all_factor;
    A q_factor;
};

// `st`: maximum and sum 2^((x - max) * kappa) of the entries that are not listed (with a tail) or of the whole row
// (without). `xc`: the student's logit at this lane's entry (-inf: none). All lanes of a warp call this together; LPR lanes belong to a row.
template <int LPR, bool TAIL, typename A>
__device__ __forceinline__ RowResult<A> solve_row(const RowStats<A> &st, const Entries<A> &en, A xc, A kappa, A inv_tau,
                                                  A weight, A gain, int KP)
{
    using M = Base2<A>;
    const A rest_sum = st.s;
    A all_max = st.max, all_sum = rest_sum;
    if (TAIL) {
        // a listed token counts once, however often it is named (no maximum takes up a NaN; the sum does)
        const A mine = en.first ? xc : A(-INFINITY);
        all_max = M::max_of(st.max, entry_max<LPR>(mine, KP));
        const A base = all_max == A(-INFINITY) ? A(0) : all_max;
        const A listed = entry_sum<LPR>(M::exp2_of((mine - base) * kappa), KP);
        all_sum = listed + (st.max == A(-INFINITY) ? rest_sum : rest_sum * M::exp2_of((st.max - base) * kappa));
    }
    const bool nothing = all_max == A(-INFINITY) && all_sum == all_sum;  // no finite entry: nothing to learn
    // the three logarithms at once, each in a lane of its own
    const int gl = threadIdx.x % LPR;
    const A of = gl == 0 ? (nothing ? A(1) : all_sum) : gl == 1 ? rest_sum : en.left;
    const A ln = M::ln_of(of);
    const A ln_s = __shfl_sync(0xffffffffu, ln, 0, LPR);
    A each = A(0);
    if (en.q > A(0)) each = en.q * (en.lq - log_prob_of(xc, all_max, inv_tau, ln_s));
    each = entry_sum<LPR>(each, KP);
    A q_all = en.sum_q, q_rest = A(0), p_rest = A(1);
    if (TAIL) {
        const A ln_rest = (st.max - all_max) * inv_tau + (__shfl_sync(0xffffffffu, ln, 1, LPR) - ln_s);
        const A ln_left = __shfl_sync(0xffffffffu, ln, 2, LPR);
        if (!st.nothing()) {
            q_rest = en.left;
            q_all = en.sum_q + q_rest;
            p_rest = rest_sum * M::exp2_of((st.max - all_max) * kappa) * M::ratio(A(1), all_sum);
            if (q_rest > A(0)) each += q_rest * (ln_left - ln_rest);
        }
    }
    A up = gain * weight * inv_tau;
    if (nothing) each = up = A(0);
    if (en.bad) each = up = A(NAN);
    if (ln_s != ln_s) each = A(NAN);  // (with no entry at all, a NaN logit would go unseen)
    RowResult<A> res;
    res.loss = weight == A(0) ? A(0) : weight * each;
    res.all_top = nothing ? A(0) : all_max;
    res.all_factor = nothing && !en.bad ? A(0) : M::ratio(up * q_all, all_sum);
    res.q_factor = up;
    if (TAIL) {
        // (Q p_rest - q_rest) / p_rest p_j, with p_j / p_rest taken from the rest's own sum
        res.top = st.max == A(-INFINITY) ? A(0) : st.max;
        res.factor = st.nothing() ? (en.bad ? A(NAN) : A(0)) : M::ratio(up * (q_all * p_rest - q_rest), rest_sum);
    } else {
        res.top = res.all_top, res.factor = res.all_factor;
    }
    return res;
}

// The gradient at this lane's entry, if no earlier one names the same token.
template <typename T>
__device__ __forceinline__ void write_entry(T *out, const Entries<typename Elt<T>::acc> &en, typename Elt<T>::acc xc,
                                            const RowResult<typename Elt<T>::acc> &res, typename Elt<T>::acc kappa,
                                            bool wanted)
{
    using A = typename Elt<T>::acc;
    using M = Base2<A>;
    if (wanted && en.first)
        out[en.c] = Elt<T>::from_acc(
            M::fma_of(M::exp2_of((xc - res.all_top) * kappa), res.all_factor, -res.q_factor * en.dup_q));
}

// Sum over the CTA of one double per thread, in a fixed order, in thread 0.
__device__ __forceinline__ double sum_cta(double v)
{
    __shared__ double parts[kRowThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kRowThreads / 32; ++w) v += parts[w];
    return v;
}

// Rows of at most LPR * NV vectors and at most LPR entries. Group g of a CTA takes the rows first + g, + GPC, ..
// The terms of the sum stay in registers for the gradient.
template <typename T, int LPR, int NV, int MODE, bool TAIL>
__global__ void __launch_bounds__(kRowThreads)
distill_rows_kernel(const __grid_constant__ DistillArgs<T> a, int run_len)
{
    using E = Elt<T>;
    using A = typename E::acc;
    using M = Base2<A>;
    constexpr int GPC = kRowThreads / LPR, VE = E::VE;
    constexpr unsigned kAll = 0xffffffffu;
    const int gl = threadIdx.x % LPR, group = threadIdx.x / LPR;
    const int64_t first = int64_t(blockIdx.x) * GPC * run_len + group;
    double sum = 0.0;
    // A row's weight decides whether it is read, its tokens what is read of it: both are asked for two rows ahead, the
    // logits at the tokens one row ahead, so that no load of a row waits for another.
    struct Ahead {
        A weight, value;
        int c;
    };
    auto look = [&](int step) {
        const int64_t r = first + int64_t(step) * GPC;
        Ahead h{A(0), A(-INFINITY), -1};
        if (step < run_len && r < a.n_rows) {
            h.weight = a.weight ? A(__ldg(a.weight + r)) : A(1);
            if (gl < a.K) {
                h.c = __ldg(a.index + r * a.K + gl);
                h.value = A(__ldg(a.teacher + r * a.K + gl));
            }
        }
        return h;
    };
    auto pick = [&](int step, const Ahead &h) {
        const int64_t r = first + int64_t(step) * GPC;
        return h.weight != A(0) && h.c >= 0 && h.c < a.V ? E::to_acc(__ldg(a.x + r * a.x_stride + h.c)) : A(-INFINITY);
    };
    Ahead now = look(0), next = look(1);
    A xc = pick(0, now);
    for (int step = 0; step < run_len; ++step) {
        const int64_t r = first + int64_t(step) * GPC;
        const bool active = r < a.n_rows;
        if (!__any_sync(kAll, active)) break;
        const int64_t rr = active ? r : 0;
        const A weight = now.weight;
        const bool seen = weight != A(0);  // a row without weight is not read
        const T *row = a.x + rr * a.x_stride;
        const RowVectors<T, MODE> rv(row, a.V);
        uint4 v[NV];
        rv.template load_all<LPR>(v, gl, seen);
        const A next_xc = pick(step + 1, next);
        const Ahead after = look(step + 2);
        const int c = seen ? now.c : -1;
        const A value = now.value;
        const Entries<A> en = weigh_entries<LPR, TAIL>(c, value, a.V, a.K, a.KP, a.inv_tau, gl);
        if (TAIL) {
            for (int e = 0; e < a.K; ++e) {
                const int token = __shfl_sync(kAll, en.c, e, LPR);
                const int at = rv.place(token < 0 ? 0 : token), i = at / VE;
                if (token >= 0 && i % LPR == gl) {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
                        if (i == j * LPR + gl) blank_element<T>(v[j], at % VE);
                }
            }
        }
        RowStats<A> st;
        st.clear();
#pragma unroll
        for (int j = 0; j < NV; ++j) st.max = M::max_of(st.max, E::vec_max(v[j]));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) st.max = M::max_of(st.max, __shfl_xor_sync(kAll, st.max, o));
        // A term is the same number in the sum and in the gradient, so the rounding of the shift leaves their ratio; it
        // is undone where the sum's logarithm is taken.
        const TermsAt<T> at(st.max, a.kappa);
        A term[NV][VE];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            E::unpack(v[j], term[j]);
            if (at.plain) {
#pragma unroll
                for (int k = 0; k < VE; ++k) term[j][k] = M::fma_of(term[j][k], a.kappa, -at.shift);
            } else {
#pragma unroll
                for (int k = 0; k < VE; ++k) term[j][k] = at.exponent(term[j][k], a.kappa);
            }
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                term[j][k] = M::exp2_of(term[j][k]);
                st.s += term[j][k];
            }
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) st.s += __shfl_xor_sync(kAll, st.s, o);
        const A undo = at.plain ? M::exp2_of(-M::fma_of(at.max, a.kappa, -at.shift)) : A(1);
        st.s *= undo;
        const A up = a.upstream && active ? A(__ldg(a.upstream + r * a.upstream_stride)) : A(1);
        const RowResult<A> res = solve_row<LPR, TAIL>(st, en, xc, a.kappa, a.inv_tau, weight, up * A(a.scale), a.KP);
        if (active && gl == 0) {
            if (a.row_loss) a.row_loss[r] = res.loss;
            sum += double(res.loss);
        }
        if (a.gx) {
            T *out = a.gx + rr * a.g_stride;
            const bool same = MODE != kAny || ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
            const A factor = res.factor * undo;
            if (active) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int i = j * LPR + gl;
#pragma unroll
                    for (int k = 0; k < VE; ++k) term[j][k] *= factor;
                    if (MODE == kFull || i < rv.count) rv.store(out, i, same, term[j]);
                }
            }
            __syncwarp();
            write_entry<T>(out, en, xc, res, a.kappa, seen);
        }
        now = next, next = after, xc = next_xc;
    }
    if (a.partial) {
        sum = sum_cta(sum);
        if (threadIdx.x == 0) a.partial[blockIdx.x] = sum * a.scale;
    }
}

// Rows that registers do not hold: a warp each (LANES = 32) or a CTA each (LANES = 256). Every warp holds the row's
// entries in its lanes. The sums run along the row, then the gradient does, reading the row a second time from L2.
template <typename T, int LANES, int MODE, bool TAIL>
__global__ void __launch_bounds__(kRowThreads)
distill_stream_kernel(const __grid_constant__ DistillArgs<T> a)
{
    using E = Elt<T>;
    using A = typename E::acc;
    using M = Base2<A>;
    constexpr int NV = 4, kWarps = kRowThreads / 32;
    __shared__ RowStats<A> parts[LANES == 32 ? 1 : kWarps];
    __shared__ int listed_of[LANES == 32 ? kWarps : 1][32];  // places of the listed tokens; -1: none
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int me = LANES == 32 ? lane : threadIdx.x;
    const int64_t r = LANES == 32 ? int64_t(blockIdx.x) * kWarps + warp : int64_t(blockIdx.x);
    const bool active = r < a.n_rows;
    A loss = A(0);
    if (active) {
        const A weight = a.weight ? A(__ldg(a.weight + r)) : A(1);
        const T *row = a.x + r * a.x_stride;
        T *out = a.gx ? a.gx + r * a.g_stride : nullptr;
        const RowVectors<T, MODE> rv(row, a.V);
        const bool same = MODE != kAny || ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
        const bool seen = weight != A(0);  // a row without weight is not read
        int c = -1;
        A value = A(-INFINITY);
        if (seen && lane < a.K) {
            c = __ldg(a.index + r * a.K + lane);
            value = A(__ldg(a.teacher + r * a.K + lane));
        }
        int *const listed = listed_of[LANES == 32 ? warp : 0];
        const A xc = c >= 0 && c < a.V ? E::to_acc(__ldg(row + c)) : A(-INFINITY);
        const Entries<A> en = weigh_entries<32, TAIL>(c, value, a.V, a.K, a.KP, a.inv_tau, lane);
        if (me < 32) listed[lane] = en.c >= 0 ? rv.place(en.c) : -1;
        if (LANES == 32)
            __syncwarp();
        else
            __syncthreads();

        // the next of this lane's vectors, from vector `from` on, that holds a listed token
        auto next_listed = [&](int from) {
            int next = 0x7fffffff;
            for (int e = 0; e < a.K; ++e) {
                const int i = listed[e] / E::VE;
                if (listed[e] >= 0 && i % LANES == me && i >= from && i < next) next = i;
            }
            return next;
        };
        RowStats<A> st;
        st.clear();
        if (seen) {
            int next = TAIL ? next_listed(0) : 0x7fffffff;
            rv.template sweep<LANES>(me, true, [&](int at, uint4(&v)[NV]) {
                if (TAIL && next < at + NV * LANES) {
                    const int past = at + NV * LANES;
                    for (int e = 0; e < a.K; ++e) {
                        const int i = listed[e] / E::VE;
                        if (listed[e] < 0 || i % LANES != me || i < at || i >= past) continue;
#pragma unroll
                        for (int j = 0; j < NV; ++j)
                            if (i == at + j * LANES) blank_element<T>(v[j], listed[e] % E::VE);
                    }
                    next = next_listed(past);
                }
                A m = st.max;
#pragma unroll
                for (int j = 0; j < NV; ++j) m = M::max_of(m, E::vec_max(v[j]));
                if (m > st.max) st.template raise<false>(m, a.kappa);
                const TermsAt<T> terms(st.max, a.kappa);
#pragma unroll
                for (int j = 0; j < NV; ++j) add_terms<T, false>(v[j], a.kappa, terms, st.s, st.t);
            });
        }
        join_lanes<32, false>(st, a.kappa);
        if (LANES > 32) {  // the warps' parts, joined in their order: the same bits in every thread
            if (lane == 0) parts[warp] = st;
            __syncthreads();
            st = parts[0];
#pragma unroll 1
            for (int w = 1; w < kWarps; ++w) st.template join<false>(parts[w], a.kappa);
        }
        st.s = st.sum(a.kappa);
        const A up = a.upstream ? A(__ldg(a.upstream + r * a.upstream_stride)) : A(1);
        const RowResult<A> res = solve_row<32, TAIL>(st, en, xc, a.kappa, a.inv_tau, weight, up * A(a.scale), a.KP);
        loss = res.loss;
        if (me == 0 && a.row_loss) a.row_loss[r] = loss;
        if (out) {
            rv.template sweep<LANES>(me, seen, [&](int at, uint4(&v)[NV]) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int i = at + j * LANES;
                    if (i < rv.count) {
                        A e[E::VE];
                        E::unpack(v[j], e);
#pragma unroll
                        for (int k = 0; k < E::VE; ++k) e[k] = M::exp2_of((e[k] - res.top) * a.kappa) * res.factor;
                        rv.store(out, i, same, e);
                    }
                }
            });
            if (LANES == 32)
                __syncwarp();
            else
                __syncthreads();
            if (me < 32) write_entry<T>(out, en, xc, res, a.kappa, seen);
        }
    }
    if (a.partial) {
        const double sum = sum_cta(me == 0 ? double(loss) : 0.0);
        if (threadIdx.x == 0) a.partial[blockIdx.x] = sum * a.scale;
    }
}

// The CTAs' sums, added up in a fixed order.
template <typename C>
__global__ void __launch_bounds__(1024) distill_sum_kernel(const double *__restrict__ partial, int64_t n, C *loss)
{
    __shared__ double parts[32];
    double v = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) v += partial[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        v = 0.0;
        for (int w = 0; w < 32; ++w) v += parts[w];
        *loss = C(v);
    }
}

template <typename T, int LPR, int NV, bool ALIGNED>
int64_t launch_distill_rows(const DistillArgs<T> &a, bool tail, cudaStream_t s)
{
    constexpr int GPC = kRowThreads / LPR;
    // runs of rows where there are enough for every SM: the first row of a run has nothing asked for ahead
    const int run_len = a.n_rows > int64_t(GPC) * kNumSMs * 32 ? 8 : 1;
    const int64_t grid = (a.n_rows + int64_t(GPC) * run_len - 1) / (int64_t(GPC) * run_len);
    auto go = [&](auto kernel) { kernel<<<unsigned(grid), kRowThreads, 0, s>>>(a, run_len); };
    if constexpr (ALIGNED) {
        if (a.V == LPR * NV * Elt<T>::VE)
            tail ? go(distill_rows_kernel<T, LPR, NV, kFull, true>) : go(distill_rows_kernel<T, LPR, NV, kFull, false>);
        else
            tail ? go(distill_rows_kernel<T, LPR, NV, kAligned, true>)
                 : go(distill_rows_kernel<T, LPR, NV, kAligned, false>);
    } else {
        tail ? go(distill_rows_kernel<T, LPR, NV, kAny, true>) : go(distill_rows_kernel<T, LPR, NV, kAny, false>);
    }
    return grid;
}

template <typename T, int LANES, bool ALIGNED>
int64_t launch_distill_stream(const DistillArgs<T> &a, bool tail, cudaStream_t s)
{
    constexpr int rows = kRowThreads / LANES, MODE = ALIGNED ? kAligned : kAny;
    const int64_t grid = (a.n_rows + rows - 1) / rows;
    if (tail)
        distill_stream_kernel<T, LANES, MODE, true><<<unsigned(grid), kRowThreads, 0, s>>>(a);
    else
        distill_stream_kernel<T, LANES, MODE, false><<<unsigned(grid), kRowThreads, 0, s>>>(a);
    return grid;
}

// Returns the number of CTAs (= sums left in a.partial).
template <typename T, bool ALIGNED>
int64_t launch_distill_t(const DistillArgs<T> &a, bool tail, cudaStream_t s)
{
    constexpr int VE = Elt<T>::VE, NV = 64 / VE < 16 ? 64 / VE : 16;
    const int nv = ALIGNED ? a.V / VE : (a.V + 2 * VE - 2) / VE;
    // Few lanes a row, many elements a lane: what a row costs beside its elements (about 400 instructions of a warp) is
    // shared by the rows of a warp. 64 elements a lane is what registers hold; every entry has a lane.
    if constexpr (sizeof(T) <= 4) {
        if (nv <= 4 * NV && a.K <= 4) return launch_distill_rows<T, 4, NV, ALIGNED>(a, tail, s);
        if (nv <= 8 * NV && a.K <= 8) return launch_distill_rows<T, 8, NV, ALIGNED>(a, tail, s);
        if (nv <= 16 * NV && a.K <= 16) return launch_distill_rows<T, 16, NV, ALIGNED>(a, tail, s);
        if (nv <= 64) return launch_distill_rows<T, 32, 2, ALIGNED>(a, tail, s);
        if (nv <= 128) return launch_distill_rows<T, 32, 4, ALIGNED>(a, tail, s);
    }
    if (nv <= 32 * NV) return launch_distill_rows<T, 32, NV, ALIGNED>(a, tail, s);
    // a warp carries a longer row where there are rows enough for the SMs' warps
    if (nv <= 2048 && a.n_rows >= kNumSMs * 32) return launch_distill_stream<T, 32, ALIGNED>(a, tail, s);
    return launch_distill_stream<T, kRowThreads, ALIGNED>(a, tail, s);
}

template <typename T>
cudaError_t launch_distill_of(const cwrnnt_rows &p, bool tail, const void *x, const void *teacher,
                              const int32_t *index, const void *weight, const void *upstream, int32_t upstream_stride,
                              double scale, double *partial, void *row_loss, void *loss, void *gx, cudaStream_t s)
{
    using C = typename Elt<T>::cost;
    constexpr int VE = Elt<T>::VE;
    DistillArgs<T> a{};
    a.x = static_cast<const T *>(x), a.gx = static_cast<T *>(gx);
    a.n_rows = p.n_rows, a.x_stride = p.x_stride, a.g_stride = p.grad_stride;
    a.V = p.V, a.K = p.n_list;
    for (a.KP = 1; a.KP < a.K;) a.KP *= 2;
    a.inv_tau = typename Elt<T>::acc(1.0 / p.temperature);
    a.kappa = typename Elt<T>::acc(kLog2e / p.temperature);
    a.scale = scale;
    a.teacher = static_cast<const C *>(teacher), a.weight = static_cast<const C *>(weight);
    a.upstream = static_cast<const C *>(upstream), a.upstream_stride = upstream_stride;
    a.index = index;
    a.row_loss = static_cast<C *>(row_loss);
    a.partial = loss ? partial : nullptr;
    auto on_boundary = [&](const void *q, int64_t stride) {
        return reinterpret_cast<uintptr_t>(q) % 16 == 0 && stride % VE == 0 && p.V % VE == 0;
    };
    const bool aligned = on_boundary(x, p.x_stride) && (!gx || on_boundary(gx, p.grad_stride));
    const int64_t sums = aligned ? launch_distill_t<T, true>(a, tail, s) : launch_distill_t<T, false>(a, tail, s);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || !loss) return e;
    distill_sum_kernel<C><<<1, 1024, 0, s>>>(partial, sums, static_cast<C *>(loss));
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_distill(const cwrnnt_rows &p, bool tail, const void *x, const void *teacher, const int32_t *index,
                           const void *weight, const void *upstream, int32_t upstream_stride, double scale,
                           double *partial, void *row_loss, void *loss, void *grad_x, cudaStream_t s)
{
    switch (p.dtype) {
    case CWRNNT_F32:
        return launch_distill_of<float>(p, tail, x, teacher, index, weight, upstream, upstream_stride, scale, partial,
                                        row_loss, loss, grad_x, s);
    case CWRNNT_F16:
        return launch_distill_of<__half>(p, tail, x, teacher, index, weight, upstream, upstream_stride, scale, partial,
                                         row_loss, loss, grad_x, s);
    case CWRNNT_BF16:
        return launch_distill_of<__nv_bfloat16>(p, tail, x, teacher, index, weight, upstream, upstream_stride, scale,
                                                partial, row_loss, loss, grad_x, s);
    case CWRNNT_F64:
        return launch_distill_of<double>(p, tail, x, teacher, index, weight, upstream, upstream_stride, scale, partial,
                                         row_loss, loss, grad_x, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace cwrnnt
