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
// Bound: HBM, 2 * V * sizeof(element) bytes a row (314340 x 1024 bf16, two entries: 0.26 ms, 5.0 TB/s; 2047 x 32003 f32,
// 32 entries: 0.135 ms, 3.9 TB/s). Rows of up to 2048 elements (1024 doubles) stay in registers between the sums
// and the gradient; longer ones take a warp or a CTA each and are read a second time, from L2 as far as they are still there:
// of 2047 x 32003 f32 rows 888 are in flight, 114 MB with their gradients on the way out, and DRAM reads come to 362 MB where
// the matrix has 262.
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
    A kappa;         // log2(e) / tau
    double inv_tau;  // 1 / tau
    double scale;    // of the summed loss and of the gradient
    const C *teacher, *weight, *upstream;
    int upstream_stride;
    bool unless_one;  // gx holds the gradient for an upstream gradient of 1 already: nothing to do if it is that
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
// ln s to the same accuracy: one step of Newton's method from the single-precision logarithm.
__device__ __forceinline__ double ln_mid(double s)
{
    const float y = logf(float(s));
    return fabsf(y) < 1e30f ? y + fma(s, exp_mid(-double(y)), -1.0) : double(y);
}
// A row's divergence is a small difference of its entries' logarithms: what is done once a row or entry is done in double.
template <typename A>
__device__ __forceinline__ double exp_of(double a)
{
    return sizeof(A) == 8 ? exp(a) : exp_mid(a);
}
template <typename A>
__device__ __forceinline__ double ln_of(double s)
{
    return sizeof(A) == 8 ? log(s) : ln_mid(s);
}

// Sums and maxima over the KP lanes (a power of two, at most `width`) that hold a row's entries, the first of the row's
// `width` lanes; the result in all of them. All lanes of a warp call these together.
template <typename V>
__device__ __forceinline__ V entry_sum(V v, int KP, int width)
{
    for (int o = KP >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return __shfl_sync(0xffffffffu, v, 0, width);
}
template <typename V>
__device__ __forceinline__ V entry_max(V v, int KP, int width)
{
    for (int o = KP >> 1; o > 0; o >>= 1) v = Base2<V>::max_of(v, __shfl_xor_sync(0xffffffffu, v, o));
    return __shfl_sync(0xffffffffu, v, 0, width);
}

// One row's teacher entry, held by lane e of `width` lanes that belong to the row, and what follows from all of them.
template <typename A>
struct Entries {
    int c;       // token, -1: none
    bool first;  // no earlier entry names the same token
    bool bad;    // some token of the row lies outside it, or the teacher gives no probability (NaN) to one
    double q, lq;  // teacher's probability and its logarithm
    A sum_q;       // over the row
    double left;   // one minus that, at least 0
    A dup_q;       // q of all entries with this token, added up in their order
};

// All lanes of a warp call this together; lane `e` of a row's lanes holds entry e: token `c`, value `a` (-1, -inf: none).
template <bool TAIL, typename A>
__device__ __forceinline__ Entries<A> weigh_entries(int c, A a, int V, int K, int KP, double inv_tau, int e, int width)
{
    constexpr unsigned kAll = 0xffffffffu;
    using M = Base2<A>;
    Entries<A> en;
    en.c = c < 0 || c >= V ? -1 : c;
    if (en.c < 0) a = A(-INFINITY);
    if (TAIL) {
        en.lq = double(a);
        en.q = exp_of<A>(en.lq);
        const double sum = entry_sum(en.q, KP, width);
        en.sum_q = A(sum);
        en.left = fmax(0.0, 1.0 - sum);
    } else {
        const double z = double(a) * inv_tau;
        const double m = entry_max(z, KP, width);
        const double w = m == -INFINITY ? 0.0 : exp_of<A>(z - m);
        const double s = entry_sum(w, KP, width);
        en.lq = s == 0.0 ? -INFINITY : z - m - ln_of<A>(s);
        en.q = s == 0.0 ? 0.0 : w / s;
        en.sum_q = s == 0.0 ? A(0) : A(s / s);
        en.left = 0.0;
    }
    const int lane = threadIdx.x & 31;
    const unsigned row = (width == 32 ? kAll : (1u << width) - 1u) << (lane / width * width);
    // (a NaN would go unseen otherwise: it compares false with everything, and fmax drops it)
    en.bad = (__ballot_sync(kAll, c >= V || a != a || (!TAIL && a == A(INFINITY))) & row) != 0;
    const unsigned same = __match_any_sync(kAll, en.c) & row;  // the row's entries with this token
    en.first = en.c >= 0 && __ffs(same) - 1 == lane;
    en.dup_q = A(en.q);
    if (__any_sync(kAll, en.c >= 0 && (same & (same - 1)) != 0)) {
        en.dup_q = A(0);
        for (int o = 0; o < K; ++o) {
            const A oq = __shfl_sync(kAll, A(en.q), o, width);
            en.dup_q += same >> (lane / width * width + o) & 1 ? oq : A(0);
        }
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

// A row's maximum and sum 2^((x - max) * kappa): of the tokens that are not listed (rest) and of all; `listed`: the listed
// tokens' part of all_sum. Without a tail rest and all are the same.
template <typename A>
struct RowSums {
    A rest_max, rest_sum, all_max, all_sum, listed;
    __device__ __forceinline__ bool nothing() const { return all_max == A(-INFINITY) && all_sum == all_sum; }
    __device__ __forceinline__ bool no_rest() const { return rest_max == A(-INFINITY) && rest_sum == rest_sum; }
};

// `mine`: the student's logit at this lane's entry if no earlier one names the token, else -inf: a listed token counts once,
// however often it is named. (No maximum takes up a NaN; the sum does.)
template <bool TAIL, typename A>
__device__ __forceinline__ RowSums<A> all_sums(A max, A sum, A mine, A kappa, int KP, int width)
{
    using M = Base2<A>;
    RowSums<A> s{max, sum, max, sum, A(0)};
    if (TAIL) {
        s.all_max = M::max_of(max, entry_max(mine, KP, width));
        const A base = s.all_max == A(-INFINITY) ? A(0) : s.all_max;
        s.listed = entry_sum(A(exp2((mine - base) * kappa)), KP, width);
        s.all_sum = s.listed + (max == A(-INFINITY) ? sum : sum * M::exp2_of((max - base) * kappa));
    }
    return s;
}

// The factors of a row's gradient, which is
//     2^((x - rest_max) * kappa) * factor                              where no entry names the token
//     2^((x - all_max) * kappa) * all_factor - q_factor * dup_q        where one does
template <typename A>
struct RowFactors {
    A rest_top, factor, all_top, all_factor, q_factor;
};
// `gain`: weight, upstream gradient, scale and 1 / tau together.
template <bool TAIL, typename A>
__device__ __forceinline__ RowFactors<A> gradient_factors(const RowSums<A> &s, A sum_q, A left, bool bad, A gain, A kappa)
{
    using M = Base2<A>;
    const bool nothing = s.nothing(), no_rest = s.no_rest();
    const A up = bad ? A(NAN) : nothing ? A(0) : gain;
    RowFactors<A> f;
    f.all_top = nothing ? A(0) : s.all_max;
    f.q_factor = up;
    const A share = nothing ? A(0) : M::ratio(A(1), s.all_sum);
    if (TAIL) {
        // (Q p_rest - q_rest) / p_rest p_j, with p_j / p_rest taken from the rest's own sum
        const A q_rest = no_rest ? A(0) : left, q_all = sum_q + q_rest;
        const A p_rest = s.rest_sum * M::exp2_of((s.rest_max - s.all_max) * kappa) * share;
        f.all_factor = up * q_all * share;
        f.rest_top = no_rest ? A(0) : s.rest_max;
        f.factor = no_rest ? (bad ? A(NAN) : A(0)) : M::ratio(up * (q_all * p_rest - q_rest), s.rest_sum);
    } else {
        f.all_factor = f.factor = up * sum_q * share;
        f.rest_top = f.all_top;
    }
    return f;
}

// A row's weighted divergence. Lane e of the row's `width` lanes holds entry e: its q, lq and the student's logit xc there.
// Both parts of the sum are joined in double: where the rest is nearly all, ln p_rest is as small as the listed tokens'
// share, and the rounding of a joined float would be all that is left of it.
template <bool TAIL, typename A>
__device__ __forceinline__ A divergence(const RowSums<A> &s, double q, double lq, A xc, double left, bool bad, A weight,
                                        double inv_tau, int KP, int width)
{
    const bool nothing = s.nothing();
    const double max = double(s.all_max);
    double all = double(s.all_sum);
    if (TAIL) all = double(s.listed) + double(s.rest_sum) * exp_of<A>((double(s.rest_max) - max) * inv_tau);
    const double ln_s = nothing ? 0.0 : ln_of<A>(all);
    double each = 0.0;
    if (q > 0.0) each = q * (lq - ((double(xc) - max) * inv_tau - ln_s));
    each = entry_sum(each, KP, width);
    if (TAIL && !s.no_rest() && left > 0.0) {
        const double ln_rest = (double(s.rest_max) - max) * inv_tau + (ln_of<A>(double(s.rest_sum)) - ln_s);
        each += left * (ln_of<A>(left) - ln_rest);
    }
    if (nothing) each = 0.0;
    if (bad || ln_s != ln_s) each = NAN;  // (with no entry at all, a NaN logit would go unseen)
    return weight == A(0) ? A(0) : A(double(weight) * each);
}

// The gradient at an entry that no earlier one names the same token as.
template <typename T>
__device__ __forceinline__ void write_entry(T *out, int c, typename Elt<T>::acc dup_q, typename Elt<T>::acc xc,
                                            const RowFactors<typename Elt<T>::acc> &f, typename Elt<T>::acc kappa)
{
    using M = Base2<typename Elt<T>::acc>;
    out[c] = Elt<T>::from_acc(M::fma_of(M::exp2_of((xc - f.all_top) * kappa), f.all_factor, -f.q_factor * dup_q));
}

// Sum over the CTA of one double per thread, in a fixed order, in thread 0.
template <int THREADS>
__device__ __forceinline__ double sum_cta(double v)
{
    __shared__ double parts[THREADS / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < THREADS / 32; ++w) v += parts[w];
    return v;
}

// What a warp keeps in shared memory of the rows that it carries: their entries, and a record each.
template <typename A>
struct EntryRecord {
    int c;    // token, -1: none
    int own;  // no earlier entry of the row names it
    A dup_q, xc;
    double q, lq;
};
template <typename A>
struct RowRecord {
    double left;
    A weight, gain, sum_q;
    RowSums<A> sums;
    int bad;
};

// Rows of at most LPR * NV vectors and at most LPR entries. Group g of a CTA takes the rows first + g, + GPC, .. run_len
// times. What a row needs beside its elements would cost a warp more instructions than the elements do, so the warp does
// that for all of its rows at once, before and after they pass: an entry to a lane. The terms of a row's sum stay in
// registers for its gradient. (314340 x 1024 bf16, two entries a row: 0.26 ms; 0.30 with that work done row by row. The
// double steps of a row are a good part of a warp's 613 instructions a row: it issues in 73 of 100 cycles.)
template <typename T, int LPR, int NV, int MODE, bool TAIL>
__global__ void __launch_bounds__(kRowThreads)
distill_rows_kernel(const __grid_constant__ DistillArgs<T> a, int run_len)
{
    using E = Elt<T>;
    using A = typename E::acc;
    using M = Base2<A>;
    constexpr int GPC = kRowThreads / LPR, VE = E::VE, kRows = 32 / LPR;  // kRows: of a warp at a time
    constexpr unsigned kAll = 0xffffffffu;
    extern __shared__ __align__(16) unsigned char scratch[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % LPR;
    const int rows = kRows * run_len, KP = a.KP;  // of this warp in all; row b is row b % kRows of step b / kRows
    RowRecord<A> *const recs = reinterpret_cast<RowRecord<A> *>(scratch) + warp * rows;
    EntryRecord<A> *const ents =
        reinterpret_cast<EntryRecord<A> *>(reinterpret_cast<RowRecord<A> *>(scratch) + kRowThreads / 32 * rows) +
        warp * rows * KP;
    if (a.unless_one && __ldg(a.upstream) == typename E::cost(1)) return;
    const int64_t first = int64_t(blockIdx.x) * GPC * run_len + warp * kRows;
    auto row_of = [&](int b) { return first + int64_t(b / kRows) * GPC + b % kRows; };

    for (int at = 0; at < rows * KP; at += 32) {
        const int i = at + lane, b = i / KP, e = i % KP;
        const int64_t r = row_of(b);
        const bool active = i < rows * KP && r < a.n_rows;
        const A weight = active ? (a.weight ? A(__ldg(a.weight + r)) : A(1)) : A(0);
        const bool seen = weight != A(0);  // a row without weight is not read
        int c = -1;
        A value = A(-INFINITY), xc = A(-INFINITY);
        if (seen && e < a.K) {
            c = __ldg(a.index + r * a.K + e);
            value = A(__ldg(a.teacher + r * a.K + e));
            if (c >= 0 && c < a.V) xc = E::to_acc(__ldg(a.x + r * a.x_stride + c));
        }
        const Entries<A> en = weigh_entries<TAIL>(c, value, a.V, a.K, KP, a.inv_tau, e, KP);
        if (i < rows * KP) {
            ents[i] = EntryRecord<A>{en.c, en.first, en.dup_q, xc, en.q, en.lq};
            if (e == 0) {
                const A up = a.upstream && active ? A(__ldg(a.upstream + r * a.upstream_stride)) : A(1);
                recs[b] = RowRecord<A>{en.left, weight, up * A(a.scale) * weight * A(a.inv_tau), en.sum_q, {}, en.bad};
            }
        }
    }
    __syncwarp();

    for (int step = 0; step < run_len; ++step) {
        const int b = step * kRows + lane / LPR;
        const int64_t r = row_of(b);
        const bool active = r < a.n_rows;
        if (!__any_sync(kAll, active)) break;
        const int64_t rr = active ? r : 0;
        RowRecord<A> &rec = recs[b];
        const EntryRecord<A> *const ent = ents + b * KP;
        const T *row = a.x + rr * a.x_stride;
        const RowVectors<T, MODE> rv(row, a.V);
        uint4 v[NV];
        rv.template load_all<LPR>(v, gl, rec.weight != A(0));
        if (TAIL) {
            for (int e = 0; e < a.K; ++e) {
                const int token = ent[e].c;
                const int at = rv.place(token < 0 ? 0 : token), i = at / VE;
                if (token >= 0 && i % LPR == gl) {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
                        if (i == j * LPR + gl) blank_element<T>(v[j], at % VE);
                }
            }
        }
        A max = A(-INFINITY), sum = A(0);
#pragma unroll
        for (int j = 0; j < NV; ++j) max = M::max_of(max, E::vec_max(v[j]));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) max = M::max_of(max, __shfl_xor_sync(kAll, max, o));
        // A term is the same number in the sum and in the gradient, so the rounding of the shift leaves their ratio; it
        // is undone where the sum stands beside another row's or its logarithm is taken.
        const TermsAt<T> at(max, a.kappa);
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
                sum += term[j][k];
            }
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
        const A undo = at.plain ? M::exp2_of(-M::fma_of(at.max, a.kappa, -at.shift)) : A(1);
        const bool holds = gl < KP && ent[gl < KP ? gl : 0].own;
        const A xc = holds ? ent[gl].xc : A(-INFINITY);
        const RowSums<A> sums = all_sums<TAIL>(max, sum * undo, xc, a.kappa, KP, LPR);
        if (gl == 0) rec.sums = sums;
        if (a.gx) {
            const RowFactors<A> f = gradient_factors<TAIL>(sums, rec.sum_q, A(rec.left), rec.bad, rec.gain, a.kappa);
            T *out = a.gx + rr * a.g_stride;
            const bool same = MODE != kAny || ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
            const A factor = f.factor * undo;
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
            if (active && holds) write_entry<T>(out, ent[gl].c, ent[gl].dup_q, xc, f, a.kappa);
        }
    }
    __syncwarp();

    double total = 0.0;
    for (int at = 0; at < rows * KP; at += 32) {
        const int i = at + lane, b = i / KP, e = i % KP;
        const bool here = i < rows * KP && row_of(b) < a.n_rows;
        const EntryRecord<A> en = here ? ents[i] : EntryRecord<A>{};
        const RowRecord<A> rec = here ? recs[b] : RowRecord<A>{};
        const A loss = divergence<TAIL>(rec.sums, en.q, en.lq, en.xc, rec.left, rec.bad, rec.weight, a.inv_tau, KP, KP);
        if (here && e == 0) {
            if (a.row_loss) a.row_loss[row_of(b)] = loss;
            total += double(loss);
        }
    }
    if (a.partial) {
        total = sum_cta<kRowThreads>(total);
        if (threadIdx.x == 0) a.partial[blockIdx.x] = total * a.scale;
    }
}

// Rows that registers do not hold: a warp each (LANES = 32) or a CTA each. Every warp holds the row's
// entries in its lanes. The sums run along the row, then the gradient does, reading the row a second time (much of it from L2).
template <typename T, int LANES, int MODE, bool TAIL>
__global__ void __launch_bounds__(LANES == 32 ? kRowThreads : LANES)
distill_stream_kernel(const __grid_constant__ DistillArgs<T> a)
{
    using E = Elt<T>;
    using A = typename E::acc;
    using M = Base2<A>;
    constexpr int NV = 4, kWarps = (LANES == 32 ? kRowThreads : LANES) / 32;
    __shared__ RowStats<A> parts[LANES == 32 ? 1 : kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int me = LANES == 32 ? lane : threadIdx.x;
    const int64_t r = LANES == 32 ? int64_t(blockIdx.x) * kWarps + warp : int64_t(blockIdx.x);
    const bool active = r < a.n_rows;
    if (a.unless_one && __ldg(a.upstream) == typename E::cost(1)) return;
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
        const A xc = c >= 0 && c < a.V ? E::to_acc(__ldg(row + c)) : A(-INFINITY);
        const Entries<A> en = weigh_entries<TAIL>(c, value, a.V, a.K, a.KP, a.inv_tau, lane, 32);
        const int place = en.c >= 0 ? rv.place(en.c) : -1;  // of this lane's entry
        RowStats<A> st;
        st.clear();
        if (seen) {
            rv.template sweep<LANES>(me, true, [&](int at, uint4(&v)[NV]) {
                if (TAIL) {  // the listed tokens among these vectors of this warp's lanes
                    const int i = place / E::VE - (at - me);
                    unsigned hits = __ballot_sync(0xffffffffu, place >= 0 && i >= 0 && i < NV * LANES &&
                                                                   (LANES == 32 || i % LANES / 32 == warp));
                    for (; hits; hits &= hits - 1) {
                        const int p = __shfl_sync(0xffffffffu, place, __ffs(hits) - 1);
#pragma unroll
                        for (int j = 0; j < NV; ++j)
                            if (p / E::VE == at + j * LANES) blank_element<T>(v[j], p % E::VE);
                    }
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
        if constexpr (LANES > 32) {
            if (lane == 0) parts[warp] = st;
            __syncthreads();
            st = join_warps<kWarps, false>(parts, a.kappa);
        }
        st.s = st.sum(a.kappa);
        const A up = a.upstream ? A(__ldg(a.upstream + r * a.upstream_stride)) : A(1);
        const RowSums<A> sums = all_sums<TAIL>(st.max, st.s, en.first ? xc : A(-INFINITY), a.kappa, a.KP, 32);
        loss = divergence<TAIL>(sums, en.q, en.lq, xc, en.left, en.bad, weight, a.inv_tau, a.KP, 32);
        if (me == 0 && a.row_loss) a.row_loss[r] = loss;
        const RowFactors<A> f =
            gradient_factors<TAIL>(sums, en.sum_q, A(en.left), en.bad, up * A(a.scale) * weight * A(a.inv_tau), a.kappa);
        if (out) {
            rv.template sweep<LANES>(me, seen, [&](int at, uint4(&v)[NV]) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int i = at + j * LANES;
                    if (i < rv.count) {
                        A e[E::VE];
                        E::unpack(v[j], e);
#pragma unroll
                        for (int k = 0; k < E::VE; ++k) e[k] = M::exp2_of((e[k] - f.rest_top) * a.kappa) * f.factor;
                        // (evict-first: the rows have to stay in L2 for this second reading, their gradients do not)
                        rv.template store<true>(out, i, same, e);
                    }
                }
            });
            if (LANES == 32)
                __syncwarp();
            else
                __syncthreads();
            if (me < 32 && en.first) write_entry<T>(out, en.c, en.dup_q, xc, f, a.kappa);
        }
    }
    if (a.partial) {
        const double sum = sum_cta<kWarps * 32>(me == 0 ? double(loss) : 0.0);
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
    using A = typename Elt<T>::acc;
    constexpr int GPC = kRowThreads / LPR;
    // runs of rows where there are enough for every SM: what is done for all rows of a warp at once needs several
    const int run_len = a.n_rows > int64_t(GPC) * kNumSMs * 32 ? 8 : 1;
    const int64_t grid = (a.n_rows + int64_t(GPC) * run_len - 1) / (int64_t(GPC) * run_len);
    // (at most 8 warps x 256 entries: K <= LPR)
    const size_t smem = size_t(GPC) * run_len * (sizeof(RowRecord<A>) + a.KP * sizeof(EntryRecord<A>));
    auto go = [&](auto kernel) {
        if (smem > 48 * 1024)
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
        kernel<<<unsigned(grid), kRowThreads, smem, s>>>(a, run_len);
    };
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
    constexpr int rows = LANES == 32 ? kRowThreads / 32 : 1, threads = LANES == 32 ? kRowThreads : LANES;
    constexpr int MODE = ALIGNED ? kAligned : kAny;
    const int64_t grid = (a.n_rows + rows - 1) / rows;
    if (tail)
        distill_stream_kernel<T, LANES, MODE, true><<<unsigned(grid), threads, 0, s>>>(a);
    else
        distill_stream_kernel<T, LANES, MODE, false><<<unsigned(grid), threads, 0, s>>>(a);
    return grid;
}

// Returns the number of CTAs (= sums left in a.partial).
template <typename T, bool ALIGNED>
int64_t launch_distill_t(const DistillArgs<T> &a, bool tail, cudaStream_t s)
{
    constexpr int VE = Elt<T>::VE, NV = 32 / VE < 16 ? 32 / VE : 16;
    const int nv = ALIGNED ? a.V / VE : (a.V + 2 * VE - 2) / VE;
    // Few lanes a row, many elements a lane: what a row costs beside its elements is shared by the rows of a warp. 32
    // elements a lane where several rows share a warp (64: 0.30 against 0.25 ms on 314340 x 1024 bf16, for want of warps);
    // every entry has a lane.
    if constexpr (sizeof(T) <= 4) {
        if (nv <= 4 * NV && a.K <= 4) return launch_distill_rows<T, 4, NV, ALIGNED>(a, tail, s);
        if (nv <= 8 * NV && a.K <= 8) return launch_distill_rows<T, 8, NV, ALIGNED>(a, tail, s);
        if (nv <= 16 * NV && a.K <= 16) return launch_distill_rows<T, 16, NV, ALIGNED>(a, tail, s);
        if (nv <= 64) return launch_distill_rows<T, 32, 2, ALIGNED>(a, tail, s);
        if (nv <= 128) return launch_distill_rows<T, 32, 4, ALIGNED>(a, tail, s);
        if (nv <= 32 * 64 / VE) return launch_distill_rows<T, 32, 64 / VE, ALIGNED>(a, tail, s);
    }
    if (nv <= 32 * NV) return launch_distill_rows<T, 32, NV, ALIGNED>(a, tail, s);
    // a warp carries a longer row where there are rows enough for the SMs' warps
    if (nv <= 2048 && a.n_rows >= kNumSMs * 32) return launch_distill_stream<T, 32, ALIGNED>(a, tail, s);
    // a CTA carries it otherwise; a larger one only where SMs would stay empty (2047 x 32003 f32: 0.19 against 0.17 ms)
    if (nv > 1024 && a.n_rows <= kNumSMs) return launch_distill_stream<T, kFewRowLanes, ALIGNED>(a, tail, s);
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
    a.inv_tau = 1.0 / p.temperature;
    a.kappa = typename Elt<T>::acc(kLog2e / p.temperature);
    a.scale = scale;
    a.teacher = static_cast<const C *>(teacher), a.weight = static_cast<const C *>(weight);
    a.upstream = static_cast<const C *>(upstream), a.upstream_stride = upstream_stride == 1 ? 1 : 0;
    a.unless_one = upstream_stride == CWRNNT_UPSTREAM_UNLESS_ONE;
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
