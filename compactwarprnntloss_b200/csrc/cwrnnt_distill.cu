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
    int V, K;
    A kappa;         // log2(e) / tau
    double inv_tau;  // 1 / tau
    double scale;    // of the summed loss and of the gradient
    const C *teacher, *weight, *upstream;
    int upstream_stride;
    const int32_t *index;
    C *row_loss;
    double *partial;  // one sum per CTA
};

// One row's teacher entry, held by lane e of the row's lanes, and what follows from all of them.
struct Entries {
    int c;           // token, -1: none
    bool first;      // no earlier entry names the same token
    double q, lq;    // teacher's probability and its logarithm
    double sum_q;    // over the row
    bool bad;        // some token of the row lies outside it
};

// All lanes of a warp call this together; LPR lanes belong to a row, lane `gl` of them holds entry gl.
template <int LPR, bool TAIL, typename C>
__device__ __forceinline__ Entries load_entries(const C *teacher, const int32_t *index, int V, int K, double inv_tau,
                                                int64_t r, int gl, bool active)
{
    constexpr unsigned kAll = 0xffffffffu;
    Entries en;
    en.c = -1;
    double a = -INFINITY;
    if (active && gl < K) {
        en.c = __ldg(index + r * K + gl);
        a = double(__ldg(teacher + r * K + gl));
    }
    const unsigned outside = __ballot_sync(kAll, en.c >= V);
    en.bad = ((outside >> ((threadIdx.x & 31) / LPR * LPR)) & (LPR == 32 ? kAll : (1u << (LPR & 31)) - 1u)) != 0;
    if (en.c >= V || en.c < 0) en.c = -1;
    en.first = en.c >= 0;
    for (int o = 0; o < K; ++o) {
        const int other = __shfl_sync(kAll, en.c, o, LPR);
        if (o < gl && other == en.c) en.first = false;
    }
    if (en.c < 0) a = -INFINITY;
    if (TAIL) {
        en.lq = a;
        en.q = exp(a);
    } else {
        const double z = a * inv_tau;
        double m = z;
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(kAll, m, o));
        const double w = m == -INFINITY ? 0.0 : exp(z - m);
        double s = w;
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
        en.lq = s == 0.0 ? -INFINITY : z - m - log(s);
        en.q = s == 0.0 ? 0.0 : w / s;
    }
    en.sum_q = en.q;
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) en.sum_q += __shfl_xor_sync(kAll, en.sum_q, o);
    return en;
}

// Element c of a vector becomes -inf.
template <typename T>
__device__ __forceinline__ void blank_element(uint4 &v, int c)
{
    using E = Elt<T>;
    typename E::acc e[E::VE];
    E::unpack(v, e);
#pragma unroll
    for (int k = 0; k < E::VE; ++k)
        if (k == c) e[k] = typename E::acc(-INFINITY);
    v = E::pack(e);
}

// What the row's statistics and entries give: its divergence, and its gradient's factors. The gradient is
//     2^((x - top) * kappa - low) * factor                                    where no entry names the token
//     2^((x - all_top) * kappa - all_low) * all_factor - q_factor * its q     where one does
template <typename A>
struct RowResult {
    double loss;  // weighted
    A top, low, factor;
    A all_top, all_low, all_factor;
    double q_factor;
};

// `st`: statistics of the entries that are not listed (with a tail) or of the whole row (without). `xc`: the student's
// logit at this lane's entry (-inf: none). All lanes of a warp call this together; LPR lanes belong to a row.
template <int LPR, bool TAIL, typename A>
__device__ __forceinline__ RowResult<A> solve_row(const RowStats<A> &st, const Entries &en, A xc, A kappa,
                                                  double inv_tau, double weight, double gain)
{
    constexpr unsigned kAll = 0xffffffffu;
    using M = Base2<A>;
    RowStats<A> all = st;
    if (TAIL) {
        RowStats<A> mine;  // a listed token counts once, however often it is named
        mine.clear();
        if (en.first && xc != A(-INFINITY)) {
            const A shift = RowStats<A>::shift_of(xc, kappa);
            mine.max = xc == xc ? xc : A(-INFINITY);  // (no maximum takes up a NaN; the sum does)
            mine.s = RowStats<A>::extreme(shift) ? xc - xc + A(1) : M::exp2_of(M::fma_of(xc, kappa, -shift));
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) {
            RowStats<A> other;
            other.max = __shfl_xor_sync(kAll, mine.max, o);
            other.s = __shfl_xor_sync(kAll, mine.s, o);
            other.t = A(0);
            mine.template join<false>(other, kappa);
        }
        all.template join<false>(mine, kappa);
    }
    const bool nothing = all.nothing();  // the student's row has no finite entry: nothing to learn
    const double log2_s = nothing ? 0.0 : all.log2_sum(kappa);
    const double ln_s = kLn2 * log2_s, max = double(all.max);
    double each = 0.0;
    if (en.q > 0.0) each = en.q * (en.lq - log_prob_of(xc, max, inv_tau, ln_s));
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) each += __shfl_xor_sync(kAll, each, o);
    double q_all = en.sum_q, q_rest = 0.0, p_rest = 1.0, rest2_s = log2_s;
    if (TAIL && !st.nothing()) {
        rest2_s = st.log2_sum(kappa);
        const double ln_rest = (double(st.max) - max) * inv_tau + kLn2 * rest2_s - ln_s;
        q_rest = fmax(0.0, 1.0 - en.sum_q);
        q_all += q_rest;
        p_rest = exp(ln_rest);
        if (q_rest > 0.0) each += q_rest * (log(q_rest) - ln_rest);
    }
    double up = gain * weight * inv_tau;
    if (nothing) each = up = 0.0;
    if (en.bad) each = up = NAN;
    if (ln_s != ln_s) each = NAN;  // (with no entry at all, a NaN logit would go unseen)
    RowResult<A> res;
    res.loss = weight == 0.0 ? 0.0 : weight * each;
    // the logarithms are rounded to the arithmetic type; the factors undo that
    res.all_top = nothing ? A(0) : all.max;
    res.all_low = A(log2_s);
    res.all_factor = A(up * q_all * exp2(double(res.all_low) - log2_s));
    res.q_factor = up;
    if (TAIL) {
        res.top = st.nothing() ? A(0) : st.max;
        res.low = A(rest2_s);
        res.factor = A(up * (q_all * p_rest - q_rest) * exp2(double(res.low) - rest2_s));
    } else {
        res.top = res.all_top, res.low = res.all_low, res.factor = res.all_factor;
    }
    return res;
}

// The gradient at this lane's entry, if no earlier one names the same token: `q` of all entries that do, added up.
template <int LPR, typename T>
__device__ __forceinline__ void write_entry(T *out, const Entries &en, typename Elt<T>::acc xc,
                                            const RowResult<typename Elt<T>::acc> &res, typename Elt<T>::acc kappa,
                                            int K, bool wanted)
{
    using A = typename Elt<T>::acc;
    using M = Base2<A>;
    double q = 0.0;
    for (int o = 0; o < K; ++o) {
        const int other = __shfl_sync(0xffffffffu, en.c, o, LPR);
        const double oq = __shfl_sync(0xffffffffu, en.q, o, LPR);
        if (other == en.c) q += oq;
    }
    if (wanted && en.first)
        out[en.c] = Elt<T>::from_acc(A(double(M::exp2_of(M::fma_of(xc - res.all_top, kappa, -res.all_low))) *
                                           double(res.all_factor) - res.q_factor * q));
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
template <typename T, int LPR, int NV, bool ALIGNED, bool TAIL>
__global__ void __launch_bounds__(kRowThreads)
distill_rows_kernel(const DistillArgs<T> a, int run_len)
{
    using E = Elt<T>;
    using A = typename E::acc;
    using M = Base2<A>;
    constexpr int GPC = kRowThreads / LPR;
    constexpr unsigned kAll = 0xffffffffu;
    const int gl = threadIdx.x % LPR, group = threadIdx.x / LPR;
    const int64_t first = int64_t(blockIdx.x) * GPC * run_len + group;
    double sum = 0.0;
    for (int step = 0; step < run_len; ++step) {
        const int64_t r = first + int64_t(step) * GPC;
        const bool active = r < a.n_rows;
        if (!__any_sync(kAll, active)) break;
        const int64_t rr = active ? r : 0;
        const double weight = active ? (a.weight ? double(__ldg(a.weight + r)) : 1.0) : 0.0;
        const bool seen = active && weight != 0.0;  // a row without weight is not read
        const T *row = a.x + rr * a.x_stride;
        const RowVectors<T, ALIGNED> rv(row, a.V);
        uint4 v[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            v[j] = vector_of_nothing<T>();
            if (seen && j * LPR + gl < rv.count) v[j] = rv.load(j * LPR + gl);
        }
        const Entries en = load_entries<LPR, TAIL>(a.teacher, a.index, a.V, a.K, a.inv_tau, rr, gl, seen);
        const A xc = en.c >= 0 ? E::to_acc(__ldg(row + en.c)) : A(-INFINITY);
        if (TAIL) {
            for (int e = 0; e < a.K; ++e) {
                const int c = __shfl_sync(kAll, en.c, e, LPR);
                const int at = c + rv.head, i = at / E::VE;
                if (c >= 0 && i % LPR == gl) {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
                        if (i == j * LPR + gl) blank_element<T>(v[j], at % E::VE);
                }
            }
        }
        RowStats<A> st;
        st.clear();
#pragma unroll
        for (int j = 0; j < NV; ++j) st.max = M::max_of(st.max, E::vec_max(v[j]));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) st.max = M::max_of(st.max, __shfl_xor_sync(kAll, st.max, o));
        const A shift = RowStats<A>::shift_of(st.max, a.kappa);
#pragma unroll
        for (int j = 0; j < NV; ++j) add_terms<T, false>(v[j], a.kappa, st.max, shift, st.s, st.t);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) st.s += __shfl_xor_sync(kAll, st.s, o);
        const double up = a.upstream && active ? double(__ldg(a.upstream + r * a.upstream_stride)) : 1.0;
        const RowResult<A> res = solve_row<LPR, TAIL>(st, en, xc, a.kappa, a.inv_tau, weight, up * a.scale);
        if (active && gl == 0) {
            if (a.row_loss) a.row_loss[r] = typename E::cost(res.loss);
            sum += res.loss;
        }
        if (a.gx) {
            T *out = a.gx + rr * a.g_stride;
            const bool same = ALIGNED || ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int i = j * LPR + gl;
                if (active && i < rv.count) {
                    A e[E::VE];
                    E::unpack(v[j], e);
#pragma unroll
                    for (int c = 0; c < E::VE; ++c)
                        e[c] = M::exp2_of(M::fma_of(e[c] - res.top, a.kappa, -res.low)) * res.factor;
                    store_vector(out, rv, i, same, e);
                }
            }
            __syncwarp();
            write_entry<LPR, T>(out, en, xc, res, a.kappa, a.K, seen);
        }
    }
    if (a.partial) {
        sum = sum_cta(sum);
        if (threadIdx.x == 0) a.partial[blockIdx.x] = sum * a.scale;
    }
}

// Any row: one CTA each. Every warp holds the row's entries in its lanes.
template <typename T, bool ALIGNED, bool TAIL>
__global__ void __launch_bounds__(kRowThreads)
distill_long_kernel(const DistillArgs<T> a)
{
    using E = Elt<T>;
    using A = typename E::acc;
    using M = Base2<A>;
    constexpr int NV = 4, kWarps = kRowThreads / 32;
    __shared__ RowStats<A> parts[kWarps];
    __shared__ int listed[32];  // positions of the listed tokens, counted from the first vector's start; -1: none
    const int tid = threadIdx.x, lane = tid & 31;
    const int64_t r = blockIdx.x;
    const double weight = a.weight ? double(__ldg(a.weight + r)) : 1.0;
    const T *row = a.x + r * a.x_stride;
    T *out = a.gx ? a.gx + r * a.g_stride : nullptr;
    const RowVectors<T, ALIGNED> rv(row, a.V);
    const bool same = ALIGNED || ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const bool seen = weight != 0.0;  // a row without weight is not read
    const Entries en = load_entries<32, TAIL>(a.teacher, a.index, a.V, a.K, a.inv_tau, r, lane, seen);
    const A xc = en.c >= 0 ? E::to_acc(__ldg(row + en.c)) : A(-INFINITY);
    if (tid < 32) listed[tid] = en.c >= 0 ? en.c + rv.head : -1;
    __syncthreads();

    // the next of this thread's vectors, from vector `from` on, that holds a listed token
    auto next_listed = [&](int from) {
        int next = 0x7fffffff;
        for (int e = 0; e < a.K; ++e) {
            const int i = listed[e] / E::VE;
            if (listed[e] >= 0 && i % kRowThreads == tid && i >= from && i < next) next = i;
        }
        return next;
    };
    RowStats<A> st;
    st.clear();
    if (seen) {
        int next = TAIL ? next_listed(0) : 0x7fffffff;
        for (int at = 0; at < rv.count; at += kRowThreads * NV) {
            uint4 v[NV];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int i = at + j * kRowThreads + tid;
                v[j] = i < rv.count ? rv.load(i) : vector_of_nothing<T>();
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int i = at + j * kRowThreads + tid;
                if (TAIL && i == next) {
                    for (int e = 0; e < a.K; ++e)
                        if (listed[e] >= 0 && listed[e] / E::VE == i) blank_element<T>(v[j], listed[e] % E::VE);
                    next = next_listed(i + 1);
                }
            }
            A m = st.max;
#pragma unroll
            for (int j = 0; j < NV; ++j) m = M::max_of(m, E::vec_max(v[j]));
            if (m > st.max) st.template raise<false>(m, a.kappa);
            const A shift = RowStats<A>::shift_of(st.max, a.kappa);
#pragma unroll
            for (int j = 0; j < NV; ++j) add_terms<T, false>(v[j], a.kappa, st.max, shift, st.s, st.t);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        RowStats<A> other;
        other.max = __shfl_xor_sync(0xffffffffu, st.max, o);
        other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
        other.t = A(0);
        st.template join<false>(other, a.kappa);
    }
    if (lane == 0) parts[tid >> 5] = st;
    __syncthreads();
    st = parts[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) st.template join<false>(parts[w], a.kappa);
    const double up = a.upstream ? double(__ldg(a.upstream + r * a.upstream_stride)) : 1.0;
    const RowResult<A> res = solve_row<32, TAIL>(st, en, xc, a.kappa, a.inv_tau, weight, up * a.scale);
    if (tid == 0) {
        if (a.row_loss) a.row_loss[r] = typename E::cost(res.loss);
        if (a.partial) a.partial[r] = res.loss * a.scale;
    }
    if (!out) return;
    for (int at = 0; at < rv.count; at += kRowThreads * NV) {
        uint4 v[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = at + j * kRowThreads + tid;
            v[j] = seen && i < rv.count ? rv.load(i) : vector_of_nothing<T>();
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = at + j * kRowThreads + tid;
            if (i < rv.count) {
                A e[E::VE];
                E::unpack(v[j], e);
#pragma unroll
                for (int c = 0; c < E::VE; ++c) e[c] = M::exp2_of(M::fma_of(e[c] - res.top, a.kappa, -res.low)) * res.factor;
                store_vector(out, rv, i, same, e);
            }
        }
    }
    __syncthreads();
    if (tid < 32) write_entry<32, T>(out, en, xc, res, a.kappa, a.K, seen);
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
    const int run_len = 1;
    const int64_t grid = (a.n_rows + int64_t(GPC) * run_len - 1) / (int64_t(GPC) * run_len);
    if (tail)
        distill_rows_kernel<T, LPR, NV, ALIGNED, true><<<unsigned(grid), kRowThreads, 0, s>>>(a, run_len);
    else
        distill_rows_kernel<T, LPR, NV, ALIGNED, false><<<unsigned(grid), kRowThreads, 0, s>>>(a, run_len);
    return grid;
}

// Returns the number of CTAs (= sums left in a.partial).
template <typename T, bool ALIGNED>
int64_t launch_distill_t(const DistillArgs<T> &a, bool tail, cudaStream_t s)
{
    constexpr int VE = Elt<T>::VE;
    const int nv = ALIGNED ? a.V / VE : (a.V + 2 * VE - 2) / VE;
    if (nv <= 16 && a.K <= 4) return launch_distill_rows<T, 4, 4, ALIGNED>(a, tail, s);
    if (nv <= 32 && a.K <= 8) return launch_distill_rows<T, 8, 4, ALIGNED>(a, tail, s);
    if (nv <= 64 && a.K <= 16) return launch_distill_rows<T, 16, 4, ALIGNED>(a, tail, s);
    if (nv <= 128) return launch_distill_rows<T, 32, 4, ALIGNED>(a, tail, s);
    if (nv <= 256) return launch_distill_rows<T, 32, 8, ALIGNED>(a, tail, s);
    if (nv <= 512) return launch_distill_rows<T, 32, 16, ALIGNED>(a, tail, s);
    if (tail)
        distill_long_kernel<T, ALIGNED, true><<<unsigned(a.n_rows), kRowThreads, 0, s>>>(a);
    else
        distill_long_kernel<T, ALIGNED, false><<<unsigned(a.n_rows), kRowThreads, 0, s>>>(a);
    return a.n_rows;
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
    a.inv_tau = 1.0 / p.temperature;
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
