// Scores of logits rows: log-probabilities of given tokens, the entropy and the largest entries of every row of a
// [n_rows, V] matrix, and the gradient of all three. With z = x / tau, lse = ln sum_j exp z_j, p_j = exp(z_j - lse):
//     log_probs[r][i]     = z[targets[r][i]] - lse
//     entropy[r]          = lse - sum_j p_j z_j
//     top_indices[r][:]   = the k largest entries, lowest index first among equals; top_log_probs[r][i] = z[...] - lse
//     grad_x[r][j]        = (1/tau) ( sum of the upstream gradients of the entries picked at j
//                                     - p_j (G + g_H (ln p_j + H)) ),   G = sum of all upstream gradients of entries
// The lattice's own gather (blank and label of every node) is the special case of two targets; here the columns are
// free, any V and any alignment is taken, and the entropy and the best alternatives come out of the same pass.
//
// Bound: HBM. Forward reads V * sizeof(element) per row, backward reads and writes that much. Rows of up to 256 vectors
// (4 KB) stay in the registers of the lanes that share them, longer ones run through a warp or a CTA each with their
// statistics alongside; the selection of the largest entries reads those again, from L1 or L2. Without a selection the
// traffic is the bound (314340 x 1024 f32, two targets and the entropy: 0.22 ms, 6.0 TB/s; its gradient 0.44 ms, 5.8
// TB/s), with one and with short rows the instructions (80003 x 4096 bf16, sixteen largest: 0.20 ms, 3.4 TB/s, 80 % of issue
// slots; 2051 x 50257 f16, twenty: 0.07 ms, 3.0 TB/s, 73 %, the second reading from L2; 600011 x 128 f16, four: 0.09 ms, 2.0
// TB/s).
//
// Selection: of the lanes' own maxima, the largest value that at least k of them reach is a lower bound of the row's
// k-th largest entry. The entries at or above it - about as many as k - are collected in shared memory and ranked by
// counting how many come before each. Rows with too many equal entries for that, rows with NaN, and long rows that a mask
// leaves fewer live lanes than the bar is taken from, are picked one entry at a time instead, by a warp that goes over the row
// for each: right, but slow (2051 x 50257 f16 with ten tokens left: eight largest 2.6 ms, twenty 6.1).
#include "cwrnnt_kernels.h"
#include "cwrnnt_rowops.cuh"

namespace cwrnnt {

namespace {

template <typename T>
struct ScoresArgs {
    using A = typename Elt<T>::acc;
    using C = typename Elt<T>::cost;
    const T *x;
    int64_t n_rows, x_stride;
    int V, n_targets, top_k;
    A kappa;    // log2(e) / tau
    A inv_tau;  // 1 / tau
    const int32_t *targets;
    C *log_probs, *entropy, *top_log_probs;
    int32_t *top_indices;
    C *stats;
};

template <typename T>
__device__ __forceinline__ void emit_top(const ScoresArgs<T> &a, const T *row, int64_t r,
                                         const RowLog<typename Elt<T>::acc> &log, int rank, int index)
{
    a.top_indices[r * a.top_k + rank] = index;
    a.top_log_probs[r * a.top_k + rank] =
        log_prob_of(Elt<T>::to_acc(__ldg(row + index)), log.max, a.inv_tau, log.ln_s);
}

// One target's log-probability: 0 where there is none (negative), NaN where it lies outside the row.
template <typename T>
__device__ __forceinline__ void emit_target(const ScoresArgs<T> &a, const T *row, int64_t r,
                                            const RowLog<typename Elt<T>::acc> &log, int t, int i)
{
    using A = typename Elt<T>::acc;
    A lp = A(0);
    if (t >= a.V)
        lp = A(NAN);
    else if (t >= 0)
        lp = log_prob_of(Elt<T>::to_acc(__ldg(row + t)), log.max, a.inv_tau, log.ln_s);
    a.log_probs[r * a.n_targets + i] = lp;
}

// Candidate keys of rows held in registers: 16-bit rows fit 32 bits (at most 256 vectors of 8 entries).
template <typename T>
struct Candidate {
    using Key = TopKey<typename Elt<T>::acc>;
    using Word = Key;
    static __device__ __forceinline__ Key of(T v, int index) { return Key::of(Elt<T>::to_acc(v), index); }
    static __device__ __forceinline__ bool before(const Key &a, const Key &b) { return a.before(b); }
    static __device__ __forceinline__ int index(const Key &k) { return k.index(); }
};
template <typename T>
struct ShortCandidate {
    using Word = uint32_t;
    static __device__ __forceinline__ uint32_t of(T v, int index) { return short_key<T>(v, index); }
    static __device__ __forceinline__ bool before(uint32_t a, uint32_t b) { return a > b; }
    static __device__ __forceinline__ int index(uint32_t k) { return int(0xffffu - (k & 0xffffu)); }
};
template <>
struct Candidate<__half> : ShortCandidate<__half> {};
template <>
struct Candidate<__nv_bfloat16> : ShortCandidate<__nv_bfloat16> {};

// (A row of fewer vectors than k has no bar, all of its entries are candidates: up to a vector for each of the lanes, which
// are at least k.)
template <typename T>
__host__ __device__ constexpr int candidates_of(int lpr)
{
    const int most = lpr * (Elt<T>::VE > 4 ? Elt<T>::VE : 4);
    return most > 32 ? most : 32;
}

// A lower bound of a row's k-th largest entry that about k entries reach: of the maxima of its lanes (of their two halves,
// where k is more than half the lanes), the smallest that fewer than k exceed. All lanes of a warp call this together.
template <int LPR, typename A>
__device__ __forceinline__ A bar_of(A early, A late, int k)
{
    constexpr unsigned kAll = 0xffffffffu;
    A bar = A(INFINITY);
    if (2 * k <= LPR) {
        const A own = Base2<A>::max_of(early, late);
        int above = 0;
#pragma unroll 8
        for (int j = 0; j < LPR; ++j) above += __shfl_sync(kAll, own, j, LPR) > own;
        if (above < k) bar = own;
    } else {
        int above0 = 0, above1 = 0;
#pragma unroll 4
        for (int j = 0; j < LPR; ++j) {
            const A o0 = __shfl_sync(kAll, early, j, LPR), o1 = __shfl_sync(kAll, late, j, LPR);
            above0 += (o0 > early) + (o1 > early);
            above1 += (o0 > late) + (o1 > late);
        }
        if (above0 < k) bar = early;
        if (above1 < k) bar = fmin(bar, late);
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) bar = fmin(bar, __shfl_xor_sync(kAll, bar, o));
    return bar;
}

// The largest entries one after the other, each by a pass over the row (from L1 or L2): for the rows of `slow` groups. Kept
// out of line, or its keys would take the registers of the usual path.
template <typename T, int LPR, int MODE>
__device__ __noinline__ void pick_one_by_one(const ScoresArgs<T> &a, const T *row, int64_t r,
                                             RowLog<typename Elt<T>::acc> log, bool slow)
{
    using Key = TopKey<typename Elt<T>::acc>;
    const int gl = threadIdx.x % LPR;
    const RowVectors<T, MODE> rv(row, a.V);
    Key last = Key::all();
    for (int round = 0; round < a.top_k; ++round) {
        Key best = Key::none();
        if (slow) {
#pragma unroll 1
            for (int i = gl; i < rv.count; i += LPR) best_after(rv, i, rv.load(i), last, best);
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) {
            const Key other = shfl_xor_key(0xffffffffu, best, o);
            if (other.before(best)) best = other;
        }
        last = best;
        if (slow && gl == 0) emit_top(a, row, r, log, round, best.index());
    }
}

// Rows of at most LPR * NV vectors: LPR lanes hold a row in NV vectors each. All lanes of a warp take every collective
// step together, whichever of their groups has a row left. Group g of a CTA takes the rows first + g, + GPC, ..
template <typename T, int LPR, int NV, int MODE, bool ENT>
__global__ void __launch_bounds__(kRowThreads)
scores_rows_kernel(const __grid_constant__ ScoresArgs<T> a, int run_len)
{
    using E = Elt<T>;
    using A = typename E::acc;
    using M = Base2<A>;
    using Cand = Candidate<T>;
    using Word = typename Cand::Word;
    constexpr int GPC = kRowThreads / LPR;
    constexpr int kCap = candidates_of<T>(LPR);
    constexpr unsigned kAll = 0xffffffffu;
    extern __shared__ __align__(16) unsigned char scratch[];  // kCap candidates per group, when top_k > 0
    const int gl = threadIdx.x % LPR, group = threadIdx.x / LPR, lane = threadIdx.x & 31;
    const unsigned group_bits = (LPR == 32 ? kAll : (1u << (LPR & 31)) - 1u) << (lane / LPR * LPR);
    Word *cands = reinterpret_cast<Word *>(scratch) + group * kCap;

    const int64_t first = int64_t(blockIdx.x) * GPC * run_len + group;
    for (int step = 0; step < run_len; ++step) {
        const int64_t r = first + int64_t(step) * GPC;
        const bool active = r < a.n_rows;
        if (!__any_sync(kAll, active)) break;
        const T *row = a.x + (active ? r : 0) * a.x_stride;
        const RowVectors<T, MODE> rv(row, a.V);
        uint4 v[NV];
        rv.template load_all<LPR>(v, gl, active);
        const int target = active && gl < a.n_targets ? __ldg(a.targets + r * a.n_targets + gl) : -1;
        A own = A(-INFINITY), own_late = A(-INFINITY);  // over the first and the second half of the lane's vectors
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (j < NV / 2)
                own = M::max_of(own, E::vec_max(v[j]));
            else
                own_late = M::max_of(own_late, E::vec_max(v[j]));
        }
        RowStats<A> st;
        st.clear();
        st.max = M::max_of(own, own_late);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) st.max = M::max_of(st.max, __shfl_xor_sync(kAll, st.max, o));
        const TermsAt<T> terms(st.max, a.kappa);
#pragma unroll
        for (int j = 0; j < NV; ++j) add_terms<T, ENT>(v[j], a.kappa, terms, st.s, st.t);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) {
            st.s += __shfl_xor_sync(kAll, st.s, o);
            if (ENT) st.t += __shfl_xor_sync(kAll, st.t, o);
        }
        const RowLog<A> log(st, a.kappa);
        if (active) {
            if (gl == 0) {
                if (ENT) a.entropy[r] = log.entropy;
                if (a.stats) a.stats[2 * r] = log.max, a.stats[2 * r + 1] = log.sum;
            }
            if (gl < a.n_targets) emit_target(a, row, r, log, target, gl);
            for (int i = gl + LPR; i < a.n_targets; i += LPR)
                emit_target(a, row, r, log, __ldg(a.targets + r * a.n_targets + i), i);
        }
        if (a.top_k > 0) {
            A bar = bar_of<LPR>(own, own_late, a.top_k);
            int n = 0;
            auto collect = [&](uint32_t bits, int j0) {
                // one candidate of every lane at a time; their places follow from the ballot
                for (;;) {
                    const unsigned have = __ballot_sync(kAll, bits != 0) & group_bits;
                    if (!__any_sync(kAll, bits != 0)) break;
                    if (bits) {
                        const int b = __ffs(bits) - 1;
                        bits &= bits - 1;
                        const int k = rv.first((j0 + b / E::VE) * LPR + gl) + b % E::VE;
                        const int at = n + __popc(have & ((1u << lane) - 1u));
                        if (at < kCap) cands[at] = Cand::of(__ldg(row + k), k);
                    }
                    n += __popc(have);
                }
            };
            constexpr int kPer = 32 / E::VE;  // vectors whose elements fit a word of bits
#pragma unroll
            for (int j0 = 0; j0 < NV; j0 += kPer) {
                uint32_t bits = 0;
#pragma unroll
                for (int j = j0; j < NV && j < j0 + kPer; ++j) {
                    const int i = j * LPR + gl;
                    uint32_t hit = at_least(rv, i, v[j], bar);
                    if (MODE != kFull && i >= rv.count) hit = 0;
                    if (!active) hit = 0;
                    bits |= hit << ((j - j0) * E::VE);
                }
                collect(bits, j0);
            }
            __syncwarp();
            const bool slow = active && (n > kCap || n < a.top_k || st.s != st.s);
            if (active && !slow) {
                for (int i = gl; i < n; i += LPR) {
                    const Word mine = cands[i];
                    int before = 0;
                    for (int j = 0; j < n; ++j) before += Cand::before(cands[j], mine);
                    if (before < a.top_k) emit_top(a, row, r, log, before, Cand::index(mine));
                }
            }
            if (__any_sync(kAll, slow)) pick_one_by_one<T, LPR, MODE>(a, row, r, log, slow);
            __syncwarp();  // the next row fills the same buffer
        }
    }
}

__host__ __device__ constexpr int stream_candidates(int lanes) { return lanes == 32 ? 96 : 512; }

// Rows that registers do not hold: a warp each (LANES = 32) or a CTA each. The statistics run along, with
// four vectors of every lane in flight. The selection reads the row again, from L1 or L2.
template <typename T, int LANES, int MODE, bool ENT>
__global__ void __launch_bounds__(LANES == 32 ? kRowThreads : LANES)
scores_stream_kernel(const __grid_constant__ ScoresArgs<T> a)
{
    using E = Elt<T>;
    using A = typename E::acc;
    using M = Base2<A>;
    using Key = TopKey<A>;
    constexpr int NV = 4, kWarps = (LANES == 32 ? kRowThreads : LANES) / 32, kCap = stream_candidates(LANES);
    constexpr int kBars = 64, kBarLanes = LANES / kBars;
    constexpr unsigned kAll = 0xffffffffu;
    extern __shared__ __align__(16) unsigned char scratch[];  // kCap keys per row of the CTA, when top_k > 0
    __shared__ RowStats<A> parts[LANES == 32 ? 1 : kWarps];
    __shared__ A bars[LANES == 32 ? 1 : kBars];
    __shared__ int counter;
    __shared__ A bar_of_row;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int me = LANES == 32 ? lane : threadIdx.x;
    const int64_t r = LANES == 32 ? int64_t(blockIdx.x) * kWarps + warp : int64_t(blockIdx.x);
    if (r >= a.n_rows) return;  // whole warps (or the CTA) leave together
    Key *const keys = reinterpret_cast<Key *>(scratch) + (LANES == 32 ? warp * kCap : 0);
    const T *row = a.x + r * a.x_stride;
    const RowVectors<T, MODE> rv(row, a.V);
    if (LANES > 32 && threadIdx.x == 0) counter = 0;

    RowStats<A> st;
    st.clear();
    A early = A(-INFINITY), late = A(-INFINITY);  // maxima over the first and the second two vectors of each four
    rv.template sweep<LANES>(me, true, [&](int, const uint4(&v)[NV]) {
        early = M::max_of(early, M::max_of(E::vec_max(v[0]), E::vec_max(v[1])));
        late = M::max_of(late, M::max_of(E::vec_max(v[2]), E::vec_max(v[3])));
        const A m = M::max_of(early, late);
        if (m > st.max) st.template raise<ENT>(m, a.kappa);
        const TermsAt<T> terms(st.max, a.kappa);
#pragma unroll
        for (int j = 0; j < NV; ++j) add_terms<T, ENT>(v[j], a.kappa, terms, st.s, st.t);
    });
    const A own = st.max;
    join_lanes<32, ENT>(st, a.kappa);
    if constexpr (LANES > 32) {
        A few = own;  // the maximum of each 64th of the lanes
#pragma unroll
        for (int o = 1; o < kBarLanes; o *= 2) few = M::max_of(few, __shfl_xor_sync(kAll, few, o));
        if (lane == 0) parts[warp] = st;
        if (lane % kBarLanes == 0) bars[threadIdx.x / kBarLanes] = few;
        __syncthreads();
        st = join_warps<kWarps, ENT>(parts, a.kappa);
    }
    const RowLog<A> log(st, a.kappa);
    if (me == 0) {
        if (ENT) a.entropy[r] = log.entropy;
        if (a.stats) a.stats[2 * r] = log.max, a.stats[2 * r + 1] = log.sum;
    }
    if (me < a.n_targets) emit_target(a, row, r, log, __ldg(a.targets + r * a.n_targets + me), me);
    if (a.top_k == 0) return;

    A bar;
    if constexpr (LANES == 32) {
        bar = bar_of<32>(early, late, a.top_k);
    } else {
        if (warp == 0) {
            bar = bar_of<32>(bars[lane], bars[lane + 32], a.top_k > 16 ? a.top_k : 17);  // of all 64
            if (lane == 0) bar_of_row = bar;
        }
        __syncthreads();
        bar = bar_of_row;
    }
    int n = 0;
    rv.template sweep<LANES>(me, true, [&](int at, const uint4(&v)[NV]) {
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = at + j * LANES;
            if (i < rv.count) bits |= at_least(rv, i, v[j], bar) << (j * E::VE);
        }
        // one candidate of every lane at a time; their places follow from the ballot
        for (;;) {
            const unsigned have = __ballot_sync(kAll, bits != 0);
            if (!have) break;
            int base = n;
            if (LANES > 32) {
                if (lane == 0) base = atomicAdd(&counter, __popc(have));
                base = __shfl_sync(kAll, base, 0);
            }
            if (bits) {
                const int b = __ffs(bits) - 1;
                bits &= bits - 1;
                const int k = rv.first(at + b / E::VE * LANES) + b % E::VE;
                const int to = base + __popc(have & ((1u << lane) - 1u));
                if (to < kCap) keys[to] = Key::of(E::to_acc(__ldg(row + k)), k);
            }
            n += __popc(have);
        }
    });
    if (LANES > 32) {
        __syncthreads();
        n = counter;
    } else {
        __syncwarp();
    }
    if (n <= kCap && n >= a.top_k && st.s == st.s) {
        for (int i = me; i < n; i += LANES) {
            const Key mine = keys[i];
            int before = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) before += keys[j].before(mine);
            if (before < a.top_k) emit_top(a, row, r, log, before, mine.index());
        }
        return;
    }
    // (uniform over the row's lanes)
    if (LANES == 32 || warp == 0) pick_one_by_one<T, 32, MODE>(a, row, r, log, true);
}

template <typename T>
struct ScoresGradArgs {
    using A = typename Elt<T>::acc;
    using C = typename Elt<T>::cost;
    const T *x;
    T *gx;
    int64_t n_rows, x_stride, g_stride;
    int V, n_targets, top_k;
    A kappa;
    double inv_tau;
    const int32_t *targets, *top_indices;
    const C *stats, *entropy, *g_log_probs, *g_entropy, *g_top;

    __device__ __forceinline__ int entries() const { return n_targets + top_k; }
    __device__ __forceinline__ int index(int64_t r, int e) const
    {
        const int t = e < n_targets ? __ldg(targets + r * n_targets + e)
                                    : __ldg(top_indices + r * top_k + (e - n_targets));
        return t < V ? t : -1;
    }
    __device__ __forceinline__ C upstream(int64_t r, int e) const
    {
        return e < n_targets ? __ldg(g_log_probs + r * n_targets + e) : __ldg(g_top + r * top_k + (e - n_targets));
    }
};

// Element-wise once the row's maximum and sum are known: LPR threads a row (a part of a warp, a warp, or a CTA), four
// vectors of each in flight. The entries that were picked are written a second time behind a barrier, by the first entry
// that names them, which adds up all that do (in their order: the sum does not depend on timing).
template <typename T, int LPR, int MODE>
__global__ void __launch_bounds__(kRowThreads)
scores_grad_kernel(const ScoresGradArgs<T> a)
{
    using E = Elt<T>;
    using A = typename E::acc;
    using M = Base2<A>;
    constexpr int NV = 4;
    constexpr int GPC = kRowThreads / LPR;
    constexpr int kSum = LPR < 32 ? LPR : 32;  // lanes that add up the entries
    const int gl = threadIdx.x % LPR;
    const int64_t r = int64_t(blockIdx.x) * GPC + threadIdx.x / LPR;
    const bool active = r < a.n_rows;
    if (LPR >= 32 && !active) return;  // whole warps (or the CTA) leave together
    const int64_t rr = active ? r : 0;
    const T *row = a.x + rr * a.x_stride;
    T *out = a.gx + rr * a.g_stride;
    const RowVectors<T, MODE> rv(row, a.V);
    const bool same = MODE != kAny || ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;

    uint4 v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if (active && j * LPR + gl < rv.count) v[j] = rv.load(j * LPR + gl);
    const int n = active ? a.entries() : 0;
    A total = A(0);
    for (int e = gl % kSum; e < n; e += kSum)
        if (a.index(rr, e) >= 0) total += a.upstream(rr, e);
#pragma unroll
    for (int o = kSum / 2; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const A max = active ? __ldg(a.stats + 2 * rr) : A(0);
    const A sum = active ? __ldg(a.stats + 2 * rr + 1) : A(1);
    const bool nothing = max == A(-INFINITY) && sum == sum;  // no finite entry: no gradient
    // p = 2^((x - top) * kappa) / sum; the row's factors carry 1 / (sum * tau)
    const A top = nothing ? A(0) : max;
    const A scale = nothing ? A(0) : A(a.inv_tau) / sum;
    A c0 = -total, c1 = A(0);
    if (a.g_entropy && active) {
        const A gh = __ldg(a.g_entropy + rr);
        c0 -= gh * (__ldg(a.entropy + rr) - (nothing ? A(0) : M::ln_of(sum)));
        c1 = -gh * A(kLn2);
    }
    c0 *= scale, c1 *= scale;
    if (nothing) c0 = c1 = A(0);  // (whatever an upstream gradient of -inf's is: zero times a NaN is none)
    if (active) {
        for (int at = 0; at < rv.count; at += LPR * NV) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int i = at + j * LPR + gl;
                if (i < rv.count) {
                    A e[E::VE];
                    E::unpack(v[j], e);
                    const int ahead = i + LPR * NV;
                    if (ahead < rv.count) v[j] = rv.load(ahead);
#pragma unroll
                    for (int c = 0; c < E::VE; ++c) {
                        const A d = (e[c] - top) * a.kappa;
                        e[c] = M::exp2_of(d) * M::fma_of(c1, M::max_of(d, M::kFloor), c0);
                    }
                    rv.store(out, i, same, e);
                }
            }
        }
    }
    if (n == 0 && LPR >= 32) return;
    if (LPR > 32)
        __syncthreads();
    else
        __syncwarp();
    for (int e = gl; e < n; e += LPR) {
        const int t = a.index(rr, e);
        if (t < 0) continue;
        A g = a.upstream(rr, e);
        bool first = true;
        if (a.n_targets > 0) {  // (the best entries differ from one another)
            g = A(0);
            for (int o = 0; o < n; ++o)
                if (a.index(rr, o) == t) {
                    g += a.upstream(rr, o);
                    first = first && o >= e;
                }
        }
        if (first) {
            const A d = (E::to_acc(__ldg(row + t)) - top) * a.kappa;
            const A own = nothing ? A(0) : g * A(a.inv_tau);
            out[t] = E::from_acc(own + M::exp2_of(d) * M::fma_of(c1, M::max_of(d, M::kFloor), c0));
        }
    }
}

// Most vectors that a row of V elements can touch.
template <typename T>
int vectors_of(int V, bool aligned)
{
    constexpr int VE = Elt<T>::VE;
    return aligned ? V / VE : (V + 2 * VE - 2) / VE;
}

template <typename T>
bool rows_aligned(const void *x, int64_t stride, int V)
{
    constexpr int VE = Elt<T>::VE;
    return reinterpret_cast<uintptr_t>(x) % 16 == 0 && stride % VE == 0 && V % VE == 0;
}

template <typename T, int LPR, int NV, bool ALIGNED>
cudaError_t launch_scores_rows(const ScoresArgs<T> &a, bool ent, cudaStream_t s)
{
    constexpr int GPC = kRowThreads / LPR;
    const int run_len = a.n_rows > int64_t(GPC) * kNumSMs * 32 ? 4 : 1;
    const int64_t grid = (a.n_rows + int64_t(GPC) * run_len - 1) / (int64_t(GPC) * run_len);
    const size_t smem = a.top_k > 0 ? GPC * candidates_of<T>(LPR) * sizeof(typename Candidate<T>::Word) : 0;
    auto go = [&](auto kernel) {
        kernel<<<unsigned(grid), kRowThreads, smem, s>>>(a, run_len);
        return cudaGetLastError();
    };
    if constexpr (ALIGNED) {
        if (a.V == LPR * NV * Elt<T>::VE)
            return ent ? go(scores_rows_kernel<T, LPR, NV, kFull, true>) : go(scores_rows_kernel<T, LPR, NV, kFull, false>);
        return ent ? go(scores_rows_kernel<T, LPR, NV, kAligned, true>)
                   : go(scores_rows_kernel<T, LPR, NV, kAligned, false>);
    }
    return ent ? go(scores_rows_kernel<T, LPR, NV, kAny, true>) : go(scores_rows_kernel<T, LPR, NV, kAny, false>);
}

template <typename T, int LANES, bool ALIGNED>
cudaError_t launch_scores_stream(const ScoresArgs<T> &a, bool ent, cudaStream_t s)
{
    constexpr int rows = LANES == 32 ? kRowThreads / 32 : 1, threads = LANES == 32 ? kRowThreads : LANES;
    constexpr int MODE = ALIGNED ? kAligned : kAny;
    const size_t smem = a.top_k > 0 ? rows * stream_candidates(LANES) * sizeof(TopKey<typename Elt<T>::acc>) : 0;
    const unsigned grid = unsigned((a.n_rows + rows - 1) / rows);
    if (ent)
        scores_stream_kernel<T, LANES, MODE, true><<<grid, threads, smem, s>>>(a);
    else
        scores_stream_kernel<T, LANES, MODE, false><<<grid, threads, smem, s>>>(a);
    return cudaGetLastError();
}

template <typename T, bool ALIGNED>
cudaError_t launch_scores_t(const ScoresArgs<T> &a, bool ent, cudaStream_t s)
{
    const int nv = vectors_of<T>(a.V, ALIGNED);
    // The bar of the selection is taken among the maxima of the lanes' halves: at least as many lanes as entries, up to a
    // warp, and no more than that, as what a row costs beside its elements is shared by the rows of a warp (600011 x 128
    // f16, four best: 112 us with 8 lanes a row, 93 with 4).
    const int lanes = a.top_k;
    if constexpr (sizeof(T) <= 4) {
        if (nv <= 16 && lanes <= 4) return launch_scores_rows<T, 4, 4, ALIGNED>(a, ent, s);
        if (nv <= 16 && lanes <= 8) return launch_scores_rows<T, 8, 2, ALIGNED>(a, ent, s);
        if (nv <= 32 && lanes <= 8) return launch_scores_rows<T, 8, 4, ALIGNED>(a, ent, s);
        if (nv <= 32 && lanes <= 16) return launch_scores_rows<T, 16, 2, ALIGNED>(a, ent, s);
        if (nv <= 64 && lanes <= 16) return launch_scores_rows<T, 16, 4, ALIGNED>(a, ent, s);
        if (nv <= 64) return launch_scores_rows<T, 32, 2, ALIGNED>(a, ent, s);
    }
    if (nv <= 128) return launch_scores_rows<T, 32, 4, ALIGNED>(a, ent, s);
    if (nv <= 256) return launch_scores_rows<T, 32, 8, ALIGNED>(a, ent, s);
    // a warp carries a longer row where there are rows enough for the SMs' warps
    if (nv <= 2048 && a.n_rows >= kNumSMs * 32) return launch_scores_stream<T, 32, ALIGNED>(a, ent, s);
    // a CTA carries it otherwise; a larger one only where SMs would stay empty (2051 x 50257 f16: 0.10 against 0.08 ms)
    if (nv > 1024 && a.n_rows <= kNumSMs) return launch_scores_stream<T, kFewRowLanes, ALIGNED>(a, ent, s);
    return launch_scores_stream<T, kRowThreads, ALIGNED>(a, ent, s);
}

template <typename T>
cudaError_t launch_scores_of(const cwrnnt_rows &p, const void *x, const int32_t *targets, void *log_probs,
                             void *entropy, void *top_log_probs, int32_t *top_indices, void *stats, cudaStream_t s)
{
    using C = typename Elt<T>::cost;
    ScoresArgs<T> a{};
    a.x = static_cast<const T *>(x);
    a.n_rows = p.n_rows, a.x_stride = p.x_stride;
    a.V = p.V, a.n_targets = p.n_list, a.top_k = p.top_k;
    a.inv_tau = typename Elt<T>::acc(1.0 / p.temperature);
    a.kappa = typename Elt<T>::acc(kLog2e / p.temperature);
    a.targets = targets;
    a.log_probs = static_cast<C *>(log_probs), a.entropy = static_cast<C *>(entropy);
    a.top_log_probs = static_cast<C *>(top_log_probs);
    a.top_indices = top_indices, a.stats = static_cast<C *>(stats);
    return rows_aligned<T>(x, p.x_stride, p.V) ? launch_scores_t<T, true>(a, entropy != nullptr, s)
                                               : launch_scores_t<T, false>(a, entropy != nullptr, s);
}

template <typename T, bool ALIGNED>
cudaError_t launch_scores_grad_t(const ScoresGradArgs<T> &a, cudaStream_t s)
{
    constexpr int kMode = ALIGNED ? kAligned : kAny;
    const int nv = vectors_of<T>(a.V, ALIGNED);
    auto grid = [&](int lpr) { return unsigned((a.n_rows + kRowThreads / lpr - 1) / (kRowThreads / lpr)); };
    if (nv <= 32)
        scores_grad_kernel<T, 8, kMode><<<grid(8), kRowThreads, 0, s>>>(a);
    else if (nv <= 1024)
        scores_grad_kernel<T, 32, kMode><<<grid(32), kRowThreads, 0, s>>>(a);
    else
        scores_grad_kernel<T, kRowThreads, kMode><<<grid(kRowThreads), kRowThreads, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_scores_grad_of(const cwrnnt_rows &p, const void *x, const int32_t *targets,
                                  const int32_t *top_indices, const void *stats, const void *entropy,
                                  const void *g_log_probs, const void *g_entropy, const void *g_top, void *gx,
                                  cudaStream_t s)
{
    using C = typename Elt<T>::cost;
    ScoresGradArgs<T> a{};
    a.x = static_cast<const T *>(x), a.gx = static_cast<T *>(gx);
    a.n_rows = p.n_rows, a.x_stride = p.x_stride, a.g_stride = p.grad_stride;
    // entries without an upstream gradient need not be looked at
    a.V = p.V, a.n_targets = g_log_probs ? p.n_list : 0, a.top_k = g_top ? p.top_k : 0;
    a.inv_tau = 1.0 / p.temperature;
    a.kappa = typename Elt<T>::acc(kLog2e / p.temperature);
    a.targets = targets, a.top_indices = top_indices;
    a.stats = static_cast<const C *>(stats), a.entropy = static_cast<const C *>(entropy);
    a.g_log_probs = static_cast<const C *>(g_log_probs), a.g_entropy = static_cast<const C *>(g_entropy);
    a.g_top = static_cast<const C *>(g_top);
    const bool aligned = rows_aligned<T>(x, p.x_stride, p.V) && rows_aligned<T>(gx, p.grad_stride, p.V);
    return aligned ? launch_scores_grad_t<T, true>(a, s) : launch_scores_grad_t<T, false>(a, s);
}

}  // namespace

cudaError_t launch_token_scores(const cwrnnt_rows &p, const void *x, const int32_t *targets, void *log_probs,
                                void *entropy, void *top_log_probs, int32_t *top_indices, void *stats, cudaStream_t s)
{
    switch (p.dtype) {
    case CWRNNT_F32:
        return launch_scores_of<float>(p, x, targets, log_probs, entropy, top_log_probs, top_indices, stats, s);
    case CWRNNT_F16:
        return launch_scores_of<__half>(p, x, targets, log_probs, entropy, top_log_probs, top_indices, stats, s);
    case CWRNNT_BF16:
        return launch_scores_of<__nv_bfloat16>(p, x, targets, log_probs, entropy, top_log_probs, top_indices, stats, s);
    case CWRNNT_F64:
        return launch_scores_of<double>(p, x, targets, log_probs, entropy, top_log_probs, top_indices, stats, s);
    }
    return cudaErrorInvalidValue;
}

cudaError_t launch_token_scores_grad(const cwrnnt_rows &p, const void *x, const int32_t *targets,
                                     const int32_t *top_indices, const void *stats, const void *entropy,
                                     const void *g_log_probs, const void *g_entropy, const void *g_top, void *grad_x,
                                     cudaStream_t s)
{
    switch (p.dtype) {
    case CWRNNT_F32:
        return launch_scores_grad_of<float>(p, x, targets, top_indices, stats, entropy, g_log_probs, g_entropy, g_top,
                                            grad_x, s);
    case CWRNNT_F16:
        return launch_scores_grad_of<__half>(p, x, targets, top_indices, stats, entropy, g_log_probs, g_entropy, g_top,
                                             grad_x, s);
    case CWRNNT_BF16:
        return launch_scores_grad_of<__nv_bfloat16>(p, x, targets, top_indices, stats, entropy, g_log_probs, g_entropy,
                                                    g_top, grad_x, s);
    case CWRNNT_F64:
        return launch_scores_grad_of<double>(p, x, targets, top_indices, stats, entropy, g_log_probs, g_entropy, g_top,
                                             grad_x, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace cwrnnt
