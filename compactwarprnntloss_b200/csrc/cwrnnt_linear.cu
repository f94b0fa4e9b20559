// The joint's linear layers on the tensor cores: y = act(x W^T + b) + r with everything but the product in its epilogue,
// and its gradients. With z = x W^T + b and dz = dy * act'(z):
//     dx = dz W,   dW = dz^T x,   db = sum over rows of dz,   dr = dy.
// Nothing but the inputs is kept for the gradients: z is multiplied out again, and the epilogue of that product writes
// dz at once (reading dy). Storing z in float instead costs more traffic than the product takes, storing it in 16 bits
// costs digits of act'(z). dz goes into its two products as the sum of two 16-bit matrices, the second what the first
// loses in its rounding: with the first alone the gradients would be off by half as much again as their own rounding. The
// second part of a float16 dz is held 2^11 times larger, or it would be below the type's range wherever dz is (upstream
// gradients of a mean over many rows): both parts together keep dz to 2^-22 of itself, and to 2^-36 where that is less. The
// tensor cores take the factor out: the second part's products are summed first, and scaled by 2^-11 as the first part's
// first product is added (40009 x 640 x 512 f16 tanh, all gradients: 5 us of 210, 3 of them for that one product of each tile,
// 2 for the factor in the epilogue).
//
// One kernel for the four products: tiles of 128 x 64 or 128 outputs, or of 256 x 256 shared by two CTAs, 64 elements of
// the sum a step. Operands come by tiled TMA into a ring of 128-byte-swizzled stages; tcgen05.mma sums in TMEM in float.
// The forward product takes both operands along the sum (K-major), dx takes W and dW takes both operands across it
// (MN-major): no operand is ever transposed in memory. Warp 0 issues the loads, warp 1 the products; four or eight more
// warps carry the previous tile out of the other half of TMEM meanwhile, through swizzled shared memory and TMA stores
// (residual and dy come the same way). CTAs are persistent; output columns run fastest, so that concurrent CTAs share
// their rows of x in L2. Products with few tiles and long sums (dW) are split along the sum; the parts are float in the
// workspace, added in a fixed order by a second kernel that carries the same epilogue.
// TMA wants rows at multiples of 16 bytes: matrices of other strides are copied to such a stride first.
//
// Bound: for large products what lies between a tile's steps (314340 x 1024 x 640 bf16: 0.36 ms, 1.14 PFLOP/s, where the
// library's bare product takes 0.34 in the same run; the tensor pipe is active 60 % of one launch's cycles, with 8.6 TB/s from
// L2) and the clock under the power limit (0.41 to 0.43 ms in a long run); with tanh or silu the epilogue's
// instructions (40009 x 640 x 512 f16: 36 us plain, 54 with tanh and residual). Sides that are no multiple of 8 cost a copy of
// their matrix, and an output of such a width leaves by 2-byte stores: 314340 x 1024 x 639 0.78 ms, 314340 x 1023 x 640 0.60.
#include "cwrnnt_kernels.h"
#include "cwrnnt_tc.cuh"

#include <cstddef>

namespace cwrnnt {

namespace {

constexpr int kBM = 128, kBK = 64;
constexpr int kMaxStages = 8;

enum { kStore = 0, kSlope = 1, kPart = 2 };

// ------------------------------------------------------------------------------------------------------- activations
__device__ __forceinline__ float rcp(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// Two elements at a time: sm_100 adds and multiplies pairs of floats in one instruction, and the epilogue of a product of
// few steps is bound by the instructions it issues (40009 x 640 x 512, an element at a time and by pairs: tanh 51 and 47 us,
// the gradient of silu 96 and 62).
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// The clamps let a NaN through.
__device__ __forceinline__ float at_least(float v, float low)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(low));
    return r;
}
__device__ __forceinline__ float at_most(float v, float high)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(high));
    return r;
}
template <int ACT>
__device__ __forceinline__ float2 activate(float2 z)
{
    if (ACT == CWRNNT_ACT_RELU) return make_float2(at_least(z.x, 0.0f), at_least(z.y, 0.0f));
    if (ACT == CWRNNT_ACT_TANH) {  // to about 2^-20 relative: 1 - 2 / (1 + e^2z), and its series where that would cancel
        const float2 m = __fmul2_rn(z, both(2.8853900817779268f));
        const float2 e = __fadd2_rn(make_float2(ex2_approx(m.x), ex2_approx(m.y)), both(1.0f));
        const float2 t = __ffma2_rn(make_float2(rcp(e.x), rcp(e.y)), both(-2.0f), both(1.0f));
        const float2 s = __fmul2_rn(z, z);
        float2 p = __ffma2_rn(s, both(-0.05396825397f), both(0.13333333333f));
        p = __ffma2_rn(s, p, both(-0.33333333333f));
        p = __ffma2_rn(__fmul2_rn(s, p), z, z);
        return make_float2(fabsf(z.x) < 0.25f ? p.x : t.x, fabsf(z.y) < 0.25f ? p.y : t.y);
    }
    if (ACT == CWRNNT_ACT_SILU) {  // below -104 the logistic function is zero in float, and so is the product
        z = make_float2(at_least(z.x, -104.0f), at_least(z.y, -104.0f));
        const float2 m = __fmul2_rn(z, both(-1.4426950408889634f));
        const float2 e = __fadd2_rn(make_float2(ex2_approx(m.x), ex2_approx(m.y)), both(1.0f));
        return __fmul2_rn(z, make_float2(rcp(e.x), rcp(e.y)));
    }
    return z;
}
// dy times the activation's slope.
template <int ACT>
__device__ __forceinline__ float2 through(float2 z, float2 dy)
{
    if (ACT == CWRNNT_ACT_RELU) {
        const float2 s = make_float2(z.x > 0.0f ? 1.0f : (z.x != z.x ? z.x : 0.0f), z.y > 0.0f ? 1.0f : (z.y != z.y ? z.y : 0.0f));
        return __fmul2_rn(dy, s);
    }
    if (ACT == CWRNNT_ACT_TANH) {  // 4 e / (1 + e)^2, e = exp(-2 |z|): no cancellation far out
        const float2 m = __fmul2_rn(z, both(2.8853900817779268f));
        const float2 e = make_float2(ex2_approx(-fabsf(m.x)), ex2_approx(-fabsf(m.y)));
        const float2 d = __fadd2_rn(e, both(1.0f)), r = make_float2(rcp(d.x), rcp(d.y));
        return __fmul2_rn(dy, __fmul2_rn(__fmul2_rn(e, r), __fmul2_rn(r, both(4.0f))));
    }
    if (ACT == CWRNNT_ACT_SILU) {  // s (1 + z (1 - s)), s the logistic function; 0 and 1 beyond -104 and 104
        z = make_float2(at_most(at_least(z.x, -104.0f), 104.0f), at_most(at_least(z.y, -104.0f), 104.0f));
        const float2 m = __fmul2_rn(z, both(-1.4426950408889634f));
        const float2 d = __fadd2_rn(make_float2(ex2_approx(m.x), ex2_approx(m.y)), both(1.0f));
        const float2 s = make_float2(rcp(d.x), rcp(d.y)), other = __ffma2_rn(s, both(-1.0f), both(1.0f));
        return __fmul2_rn(dy, __fmul2_rn(s, __ffma2_rn(z, other, both(1.0f))));
    }
    return dy;
}
template <int ACT>
__device__ __forceinline__ float2 finish_one(bool slope, float2 z, float2 side)
{
    return slope ? through<ACT>(z, side) : __fadd2_rn(activate<ACT>(z), side);
}

// ---------------------------------------------------------------------------------------------------------- epilogue
struct Epilogue {
    int mode;           // kStore, kSlope, kPart
    int act;
    const void *bias;   // [N] or null
    const void *side;   // kStore: residual [M, side_ld] or null; kSlope: dy [M, side_ld]
    void *out;          // [M, out_ld]; kPart: float [splits * rows of tiles, out_ld]
    int64_t side_ld, out_ld;
    bool tma_out;            // rows of out lie on 16-byte boundaries: they go by TMA (rows of side always do)
    bool vec;                // all 16-byte accesses allowed, columns in whole groups of 8
    float *sums;             // kSlope: sums over each 32 rows of dz, [rows / 32, N], or null
    void *low;               // kSlope: what dz loses in its rounding, scaled and rounded again, as `out`; or null
    __host__ __device__ int pieces() const { return 1 + (side != nullptr) + (low != nullptr); }
};

// What becomes of an element of the product once the bias is added: an activation, or (kSlopeOf + activation) the upstream
// gradient times the activation's slope.
constexpr int kSlopeOf = 8;
template <int KIND, bool SIDE>
__device__ __forceinline__ float2 finish(float2 v, float2 side)
{
    if constexpr (KIND >= kSlopeOf) {
        return through<KIND - kSlopeOf>(v, side);
    } else {
        v = activate<KIND>(v);
        return SIDE ? __fadd2_rn(v, side) : v;
    }
}
__device__ __forceinline__ float finish_as(const Epilogue &ep, float v, float side)
{
    const bool slope = ep.mode == kSlope;
    const float2 z = make_float2(v, 0.0f), s = make_float2(side, 0.0f);
    if (ep.act == CWRNNT_ACT_RELU) return finish_one<CWRNNT_ACT_RELU>(slope, z, s).x;
    if (ep.act == CWRNNT_ACT_TANH) return finish_one<CWRNNT_ACT_TANH>(slope, z, s).x;
    if (ep.act == CWRNNT_ACT_SILU) return finish_one<CWRNNT_ACT_SILU>(slope, z, s).x;
    return finish_one<CWRNNT_ACT_NONE>(slope, z, s).x;
}

// The low part of dz is held 2^kLowShift times larger: bfloat16 has float's range; what a float16 loses is at most 16, and
// 16 * 2^11 is in its range.
template <typename T>
constexpr int kLowShift = Elt<T>::kBf16 ? 0 : 11;
template <typename T>
constexpr float kLowScale = float(1 << kLowShift<T>);

// What v loses when it is rounded to T, scaled and rounded to T.
template <typename T>
__device__ __forceinline__ T low_part(float v)
{
    const float high = Elt<T>::to_acc(Elt<T>::from_acc(v));
    return Elt<T>::from_acc(fabsf(high) < INFINITY ? (v - high) * kLowScale<T> : 0.0f);
}

// All bits of the halves of a word that are finite.
template <typename T>
__device__ __forceinline__ uint32_t finite_mask(uint32_t w)
{
    if constexpr (Elt<T>::kBf16) {
        const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162 *>(&w);
        return __hlt2_mask(__habs2(h), __nv_bfloat162(__ushort_as_bfloat16(0x7f80), __ushort_as_bfloat16(0x7f80)));
    } else {
        const __half2 h = *reinterpret_cast<const __half2 *>(&w);
        return __hlt2_mask(__habs2(h), __half2(__ushort_as_half(0x7c00), __ushort_as_half(0x7c00)));
    }
}

// Columns [col, col + 8) of one row straight from and to global memory, `n` of them inside the matrix.
template <typename T>
__device__ __forceinline__ void finish_in_place(const Epilogue &ep, float (&v)[8], int64_t row, int col, int n)
{
    using E = Elt<T>;
    float s[8] = {};
    if (ep.bias) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
            if (c < n) v[c] += E::to_acc(__ldg(static_cast<const T *>(ep.bias) + col + c));
    }
    if (ep.side) {
        const T *side = static_cast<const T *>(ep.side) + row * ep.side_ld + col;
        if (ep.vec) {
            E::unpack(__ldg(reinterpret_cast<const uint4 *>(side)), s);
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) s[c] = c < n ? E::to_acc(__ldg(side + c)) : 0.0f;
        }
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = finish_as(ep, v[c], s[c]);
    T *out = static_cast<T *>(ep.out) + row * ep.out_ld + col;
    if (ep.vec) {
        *reinterpret_cast<uint4 *>(out) = E::pack(v);
    } else {
#pragma unroll
        for (int c = 0; c < 8; ++c)
            if (c < n) out[c] = E::from_acc(v[c]);
    }
    if (ep.low) {
        T *low = static_cast<T *>(ep.low) + row * ep.out_ld + col;
#pragma unroll
        for (int c = 0; c < 8; ++c)
            if (c < n) low[c] = low_part<T>(v[c]);
    }
}

// ------------------------------------------------------------------------------------------------------------- kernel
struct Shape {
    int64_t M;
    int N;
    int steps;       // steps of kBK along the sum, in all
    int half_steps;  // of them, those of A's low part, the first ones: A may be a matrix and a low part (0: it is one)
    int steps_per_split, splits;
    int64_t tiles_m;
    int tiles_n;
    int stages;
    int64_t part_rows;
    // columns that tile n multiplies out: the last tile of a row is as wide as the matrix needs it
    __device__ __forceinline__ int width(int n, int bn, int ctas) const
    {
        const int unit = 16 * ctas, left = (N - n * bn + unit - 1) / unit * unit;
        return left < bn ? left : bn;
    }
    __device__ __forceinline__ int64_t tiles() const { return tiles_m * tiles_n * splits; }
    // columns fastest, then rows, then parts of the sum
    __device__ __forceinline__ void tile(int64_t t, int64_t &m, int &n, int &split) const
    {
        n = int(t % tiles_n);
        t /= tiles_n;
        m = t % tiles_m;
        split = int(t / tiles_m);
    }
    __device__ __forceinline__ int first_step(int split) const { return split * steps_per_split; }
    __device__ __forceinline__ int count_steps(int split) const
    {
        const int left = steps - first_step(split);
        return left < steps_per_split ? left : steps_per_split;
    }
    // a part of the sum that holds products of the low part only
    __device__ __forceinline__ bool low_only(int split) const { return first_step(split) + count_steps(split) <= half_steps; }
};

// A warp of the epilogue carries 32 rows by pieces of 128 bytes (64 columns of 16 bits, 32 of a part's floats) through a
// buffer of its own, in the swizzle of the TMA copies: 16-byte group j of row r lies at group j ^ (r & 7), so that neither
// a thread's row nor a row of the warp meets bank conflicts.
constexpr int kPiece = 32 * 128;
constexpr int kMostCarriers = 8;

// The kernel's shared memory behind the stages and the pieces.
struct Control {
    uint64_t full[kMaxStages], empty[kMaxStages], sum_full[2], sum_empty[2], drained, side_full[kMostCarriers];
    uint32_t tmem_slot;
    int gave_up;
    float bias[kMostCarriers][64];
};
static_assert(offsetof(Control, bias) % 16 == 0, "read in vectors");
template <int BN>
struct Layout {
    // the widest tiles are shared by two CTAs: 256 rows, half of them and half of the columns' operand in each
    static constexpr bool kPair = BN == 256;
    static constexpr int kRowsB = kPair ? BN / 2 : BN;
    static constexpr int kA = kBM * kBK * 2, kB = kRowsB * kBK * 2, kStage = kA + kB;
    static constexpr int kCarriers = BN >= 128 ? 8 : 4;  // warps of the epilogue
    static constexpr int kThreads = 64 + 32 * kCarriers;
    static constexpr uint32_t kColumns = 2 * BN;         // two sums in TMEM
    // `pieces`: of each carrier, one on its way out, one in where there is a side, another out where dz has a low part
    static constexpr int stages(int pieces)
    {
        const int n = (227 * 1024 - int(sizeof(Control)) - kCarriers * kPiece * pieces) / kStage;
        return n < kMaxStages ? n : kMaxStages;
    }
    static constexpr int bytes(int pieces)
    {
        return stages(pieces) * kStage + kCarriers * kPiece * pieces + int(sizeof(Control));
    }
    static constexpr int most_bytes()
    {
        const int a = bytes(1), b = bytes(2), c = bytes(3);
        return a > b ? (a > c ? a : c) : (b > c ? b : c);
    }
};

__device__ __forceinline__ uint4 *piece_group(unsigned char *piece, int row, int group)
{
    return reinterpret_cast<uint4 *>(piece + row * 128 + ((group ^ (row & 7)) << 4));
}

// One warp's share of the tiles: 32 rows, by pieces of 64 columns (32 of a part). What a piece needs from global memory
// (upstream gradient or residual by TMA, the bias in registers) is asked for one piece ahead, and the sums are given
// back to the products as soon as they are read. The piece's arithmetic is compiled for each kind of epilogue: with
// branches between its eight-column groups two warps per scheduler could not hide its latencies (measured on the
// Conformer logits: 0.40 ms that way).
template <typename T>
struct Carrier {
    using E = Elt<T>;
    const Epilogue &ep;
    const int64_t M;
    const int N;
    const CUtensorMap *map_out, *map_side, *map_low;
    unsigned char *out_piece, *side_piece, *low_piece;
    float *bias;  // 64 of them
    uint64_t *side_bar;
    volatile int *gave_up;
    uint32_t side_phase;
    int lane;
    float next_bias[2];

    // what the piece at (row0, col) needs
    __device__ __forceinline__ void ask(int row0, int col)
    {
        if (ep.side && lane == 0) {
            tc::mbar_expect(side_bar, kPiece);
            tc::load_2d(side_piece, map_side, side_bar, col, row0);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = col + h * 32 + lane;
            next_bias[h] = ep.bias && c < N ? E::to_acc(__ldg(static_cast<const T *>(ep.bias) + c)) : 0.0f;
        }
    }
    template <int KIND, bool SIDE, typename Release>
    __device__ __forceinline__ void columns(uint32_t d, int row0, int next_col, bool ok, Release &release)
    {
        uint32_t r[2][32];
        tc::tmem_load32(d, r[0]);
        tc::tmem_load32(d + 32, r[1]);
        uint4 side[8];
        if (SIDE) {
#pragma unroll
            for (int g = 0; g < 8; ++g) side[g] = *piece_group(side_piece, lane, g);
        }
        tc::tmem_load_wait();
        __syncwarp();
        if (next_col >= 0)
            ask(row0, next_col);
        else
            release();
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            float v[8], s[8] = {};
            const float4 b0 = *reinterpret_cast<const float4 *>(bias + g * 8);
            const float4 b1 = *reinterpret_cast<const float4 *>(bias + g * 8 + 4);
            const float2 b[4] = {{b0.x, b0.y}, {b0.z, b0.w}, {b1.x, b1.y}, {b1.z, b1.w}};
            if (SIDE) E::unpack(side[g], s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t *z = &r[g / 4][g % 4 * 8 + 2 * i];
                const float2 sum = __fadd2_rn(make_float2(__uint_as_float(z[0]), __uint_as_float(z[1])), b[i]);
                const float2 f = finish<KIND, SIDE>(sum, make_float2(s[2 * i], s[2 * i + 1]));
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            }
            uint4 w = E::pack(v);
            if (!ok) w = make_uint4(~0u, ~0u, ~0u, ~0u);  // a wait that ran out leaves NaN
            *piece_group(out_piece, lane, g) = w;
            if constexpr (KIND == kSlopeOf + CWRNNT_ACT_TANH || KIND == kSlopeOf + CWRNNT_ACT_SILU) {
                E::unpack(w, s);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    float2 lost = __ffma2_rn(make_float2(s[i], s[i + 1]), both(-1.0f), make_float2(v[i], v[i + 1]));
                    if (kLowShift<T> > 0) lost = __fmul2_rn(lost, both(kLowScale<T>));
                    v[i] = lost.x, v[i + 1] = lost.y;
                }
                const uint4 low = E::pack(v);
                *piece_group(low_piece, lane, g) = make_uint4(low.x & finite_mask<T>(w.x), low.y & finite_mask<T>(w.y),
                                                              low.z & finite_mask<T>(w.z), low.w & finite_mask<T>(w.w));
            }
        }
    }
    template <typename Release>
    __device__ __forceinline__ void columns_of_part(uint32_t d, float factor, int next_col, bool ok, Release &release)
    {
        uint32_t r[32];
        tc::tmem_load32(d, r);
        tc::tmem_load_wait();
        __syncwarp();
        if (next_col < 0) release();
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            uint4 w = make_uint4(r[4 * g], r[4 * g + 1], r[4 * g + 2], r[4 * g + 3]);
            if constexpr (kLowShift<T> > 0) {
                w.x = __float_as_uint(__uint_as_float(w.x) * factor), w.y = __float_as_uint(__uint_as_float(w.y) * factor);
                w.z = __float_as_uint(__uint_as_float(w.z) * factor), w.w = __float_as_uint(__uint_as_float(w.w) * factor);
            }
            if (!ok) w = make_uint4(~0u, ~0u, ~0u, ~0u);
            *piece_group(out_piece, lane, g) = w;
        }
    }
    // The piece's first n rows added up: columns 2 * lane and 2 * lane + 1. (Rows behind the matrix are no sum of anything:
    // their upstream gradient is zero, but their z is NaN where a weight is infinite.)
    __device__ __forceinline__ void add_rows(unsigned char *piece, int n, float &s0, float &s1) const
    {
        auto add = [&](int k) {
            const uint32_t w = reinterpret_cast<const uint32_t *>(piece_group(piece, k, lane >> 2))[lane & 3];
            float v[8];
            E::unpack(make_uint4(w, 0u, 0u, 0u), v);
            s0 += v[0], s1 += v[1];
        };
        if (n == 32) {
#pragma unroll 8
            for (int k = 0; k < 32; ++k) add(k);
        } else {
#pragma unroll 1
            for (int k = 0; k < n; ++k) add(k);
        }
    }
    // `d`: TMEM address of the piece's first column in this warp's lanes; `factor`: of a part's sums; `release`: gives the
    // tile's sums back
    template <typename Release>
    __device__ __forceinline__ void piece(uint32_t d, int row0, int64_t out_row0, int col, float factor, bool ok,
                                          int next_col, Release &release)
    {
        if (ep.mode != kPart) {
            bias[lane] = next_bias[0], bias[32 + lane] = next_bias[1];
            if (ep.side) {
                ok = tc::mbar_wait(side_bar, side_phase, gave_up) && ok;
                side_phase ^= 1;
            }
        }
        if (lane == 0) tc::stores_read();  // the last piece has left the buffer
        __syncwarp();
#define CWRNNT_KIND(KIND, SIDE) columns<KIND, SIDE>(d, row0, next_col, ok, release)
        if (ep.mode == kPart) {
            columns_of_part(d, factor, next_col, ok, release);
        } else if (ep.mode == kSlope) {
            if (ep.act == CWRNNT_ACT_RELU)
                CWRNNT_KIND(kSlopeOf + CWRNNT_ACT_RELU, true);
            else if (ep.act == CWRNNT_ACT_TANH)
                CWRNNT_KIND(kSlopeOf + CWRNNT_ACT_TANH, true);
            else
                CWRNNT_KIND(kSlopeOf + CWRNNT_ACT_SILU, true);
        } else if (ep.side) {
            if (ep.act == CWRNNT_ACT_NONE)
                CWRNNT_KIND(CWRNNT_ACT_NONE, true);
            else if (ep.act == CWRNNT_ACT_RELU)
                CWRNNT_KIND(CWRNNT_ACT_RELU, true);
            else if (ep.act == CWRNNT_ACT_TANH)
                CWRNNT_KIND(CWRNNT_ACT_TANH, true);
            else
                CWRNNT_KIND(CWRNNT_ACT_SILU, true);
        } else {
            if (ep.act == CWRNNT_ACT_NONE)
                CWRNNT_KIND(CWRNNT_ACT_NONE, false);
            else if (ep.act == CWRNNT_ACT_RELU)
                CWRNNT_KIND(CWRNNT_ACT_RELU, false);
            else if (ep.act == CWRNNT_ACT_TANH)
                CWRNNT_KIND(CWRNNT_ACT_TANH, false);
            else
                CWRNNT_KIND(CWRNNT_ACT_SILU, false);
        }
#undef CWRNNT_KIND
        if (ep.tma_out) tc::fence_async();
        __syncwarp();
        if (ep.tma_out && lane == 0) {
            tc::store_2d(map_out, out_piece, col, int(out_row0));
            if (ep.low) tc::store_2d(map_low, low_piece, col, int(out_row0));
        }
        float s0 = 0.0f, s1 = 0.0f;
        const int rows = M - row0 < 32 ? int(M - row0) : 32;
        if (ep.sums) add_rows(out_piece, rows, s0, s1);
        if (ep.sums && ep.low) {
            float l0 = 0.0f, l1 = 0.0f;
            add_rows(low_piece, rows, l0, l1);
            s0 += l0 * (1.0f / kLowScale<T>), s1 += l1 * (1.0f / kLowScale<T>);
        }
        if (ep.sums) {
            float *to = ep.sums + int64_t(row0 / 32) * N + col + 2 * lane;
            if (col + 2 * lane < N) to[0] = s0;
            if (col + 2 * lane + 1 < N) to[1] = s1;
        }
        if (!ep.tma_out) {
            const T *o = reinterpret_cast<const T *>(out_piece);
            for (int k = 0; k < 32; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int c = h * 32 + lane;
                    if (row0 + k < M && col + c < N)
                        static_cast<T *>(ep.out)[int64_t(row0 + k) * ep.out_ld + col + c] =
                            o[k * 64 + (((c >> 3) ^ (k & 7)) << 3) + (c & 7)];
                }
        }
        __syncwarp();
    }
};

template <typename T, int BN, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(Layout<BN>::kThreads, 1)
linear_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
              const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_side,
              const __grid_constant__ CUtensorMap map_low,
              const __grid_constant__ Shape sh, const __grid_constant__ Epilogue ep)
{
    using L = Layout<BN>;
    // stages, pieces, control: the stages start on a 1024-byte boundary, as the swizzle wants it
    extern __shared__ __align__(1024) unsigned char stages[];
    unsigned char *const pieces = stages + sh.stages * L::kStage;
    Control &ctl = *reinterpret_cast<Control *>(pieces + L::kCarriers * kPiece * ep.pieces());
    uint64_t *const full = ctl.full, *const empty = ctl.empty;
    uint64_t *const sum_full = ctl.sum_full, *const sum_empty = ctl.sum_empty;
    const bool placed = (tc::smem_addr(stages) & 1023) == 0;  // else every role gives up at once
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr bool kPair = L::kPair;
    constexpr int kCtas = kPair ? 2 : 1;
    const int rank = kPair ? int(tc::cluster_rank()) : 0;
    const int64_t t0 = blockIdx.x / kCtas, dt = gridDim.x / kCtas;

    if (warp == 0 && lane == 0) {
        for (int i = 0; i < sh.stages; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&sum_full[i], 1);
            tc::mbar_init(&sum_empty[i], L::kCarriers * kCtas);
        }
        for (int i = 0; i < L::kCarriers; ++i) tc::mbar_init(&ctl.side_full[i], 1);
        tc::mbar_init(&ctl.drained, 1);
        ctl.gave_up = !placed;
        tc::mbar_init_fence();
        tc::prefetch_map(&map_a);
        tc::prefetch_map(&map_b);
    }
    if (warp == 1) tc::tmem_alloc<kPair>(&ctl.tmem_slot, L::kColumns);
    __syncwarp();
    tc::fence_before();
    if (kPair)
        tc::cluster_sync();
    else
        __syncthreads();
    tc::fence_after();
    const uint32_t tmem = ctl.tmem_slot;
    const int64_t total = sh.tiles();

    if (warp == 0) {
        if (lane == 0) {
            int at = 0;
            uint32_t phase = 0;
            bool ok = placed;
            uint32_t started = 0;  // stages loaded at least once
            for (int64_t t = t0; ok && t < total; t += dt) {
                int64_t m;
                int n, split;
                sh.tile(t, m, n, split);
                const int k0 = sh.first_step(split), k1 = k0 + sh.count_steps(split);
                const int row = (int(m) * kCtas + rank) * kBM;
                const int col = n * BN + rank * (sh.width(n, BN, kCtas) / 2);
                for (int t_k = k0; ok && t_k < k1; ++t_k) {
                    ok = tc::mbar_wait(&empty[at], phase ^ 1, &ctl.gave_up);
                    if (!ok) break;
                    const bool low = t_k < sh.half_steps;
                    const int k = low ? t_k : t_k - sh.half_steps;
                    const CUtensorMap *const from_a = low ? &map_low : &map_a;
                    unsigned char *a = stages + at * L::kStage, *b = a + L::kA;
                    if (rank == 0) tc::mbar_expect(&full[at], L::kStage * kCtas);
                    const uint32_t bar = kPair ? tc::peer_addr(&full[at], 0) : 0;
                    auto load = [&](unsigned char *dst, const CUtensorMap *map, int x, int y) {
                        if (kPair)
                            tc::load_2d_pair(dst, map, bar, x, y);
                        else
                            tc::load_2d(dst, map, &full[at], x, y);
                    };
                    if (A_MN) {
#pragma unroll
                        for (int i = 0; i < kBM / 64; ++i) load(a + i * 8192, from_a, row + i * 64, k * kBK);
                    } else {
                        load(a, from_a, k * kBK, row);
                    }
                    if (B_MN) {
#pragma unroll
                        for (int i = 0; i < L::kRowsB / 64; ++i) load(b + i * 8192, &map_b, col + i * 64, k * kBK);
                    } else {
                        load(b, &map_b, k * kBK, col);
                    }
                    started |= 1u << at;
                    if (++at == sh.stages) at = 0, phase ^= 1;
                }
            }
            // every load has landed before the CTA's memory goes: the last fill of each stage (of a pair, the first CTA's
            // barriers count both CTAs' loads, and the other waits for it at the end)
            for (int i = 0; rank == 0 && i < sh.stages; ++i) {
                if (!(started >> i & 1)) continue;
                const uint32_t last = i < at ? phase : phase ^ 1;
                tc::mbar_drain(&full[i], last);
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int at = 0, half = 0;
            uint32_t phase = 0, half_phase = 0;
            bool ok = placed;
            for (int64_t t = t0; ok && t < total; t += dt) {
                int64_t m;
                int n, split;
                sh.tile(t, m, n, split);
                const uint32_t idesc = tc::instruction(Elt<T>::kBf16 ? 1 : 0, A_MN, B_MN, kBM * kCtas,
                                                       sh.width(n, BN, kCtas));
                ok = tc::mbar_wait(&sum_empty[half], half_phase ^ 1, &ctl.gave_up);
                if (!ok) break;
                tc::fence_after();
                const uint32_t d = tmem + uint32_t(half * BN);
                const int steps = sh.count_steps(split);
                // the step before which the low part's sum is scaled, if there is one here (only dz has a low part: B is
                // MN-major then)
                constexpr bool kScales = kLowShift<T> > 0 && B_MN;
                const int scaled = kScales ? sh.half_steps - sh.first_step(split) : 0;
                for (int k = 0; ok && k < steps; ++k) {
                    ok = tc::mbar_wait(&full[at], phase, &ctl.gave_up);
                    if (!ok) break;
                    tc::fence_after();
                    const uint32_t a = tc::smem_addr(stages + at * L::kStage), b = a + L::kA;
                    // 16 elements of the sum: 32 bytes along a K-major row, 16 rows of an MN-major operand
                    auto operand_a = [&](int i) { return tc::operand(a + i * (A_MN ? 2048 : 32), A_MN ? 8192 : 16, 1024); };
                    auto operand_b = [&](int i) { return tc::operand(b + i * (B_MN ? 2048 : 32), B_MN ? 8192 : 16, 1024); };
                    const bool scales = kScales && k > 0 && k == scaled;
                    if (scales)
                        tc::mma_f16_scaled<kPair, kLowShift<T>>(d, operand_a(0), operand_b(0), idesc);
                    else
                        tc::mma_f16<kPair>(d, operand_a(0), operand_b(0), idesc, k > 0);
#pragma unroll
                    for (int i = 1; i < kBK / 16; ++i) tc::mma_f16<kPair>(d, operand_a(i), operand_b(i), idesc, 1);
                    tc::commit<kPair>(&empty[at]);
                    if (++at == sh.stages) at = 0, phase ^= 1;
                }
                if (ok) tc::commit<kPair>(&sum_full[half]);
                if (++half == 2) half = 0, half_phase ^= 1;
            }
            // every product has left the tensor core before the CTA's memory goes
            tc::commit<kPair>(&ctl.drained);
            tc::mbar_drain(&ctl.drained, 0);
        }
    } else {
        const int quarter = warp & 3;  // the TMEM lanes that this warp may read
        const int carrier = warp - 2, share = carrier / 4;
        constexpr int kShares = L::kCarriers / 4;
        int half = 0;
        uint32_t half_phase = 0;
        Carrier<T> c{ep, sh.M, sh.N, &map_out, &map_side, &map_low, pieces + carrier * kPiece,
                     pieces + (L::kCarriers + carrier) * kPiece, pieces + (2 * L::kCarriers + carrier) * kPiece,
                     ctl.bias[carrier], &ctl.side_full[carrier], &ctl.gave_up,
                     0, lane, {}};
        const int step = ep.mode == kPart ? 32 : 64;
        for (int64_t t = t0; t < total; t += dt) {
            int64_t m;
            int n, split;
            sh.tile(t, m, n, split);
            const int row0 = int(m * kCtas + rank) * kBM + quarter * 32;
            const int n0 = n * BN;
            const int end = n0 + BN < sh.N ? n0 + BN : sh.N;
            int col = n0 + share * step;
            const bool mine = row0 < sh.M && col < end;
            if (mine) c.ask(row0, col);
            const bool ok = tc::mbar_wait(&sum_full[half], half_phase, &ctl.gave_up);
            tc::fence_after();
            __syncwarp();
            const uint32_t d = tmem + uint32_t(half * BN) + (uint32_t(quarter * 32) << 16);
            const float factor = sh.low_only(split) ? 1.0f / kLowScale<T> : 1.0f;
            auto release = [&] {  // this half of TMEM is free for another tile's sums
                tc::fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (kPair)
                        tc::mbar_arrive_peer(tc::peer_addr(&sum_empty[half], 0));
                    else
                        tc::mbar_arrive(&sum_empty[half]);
                }
            };
            if (!mine) release();
            for (; mine && col < end; col += kShares * step) {
                const int next = col + kShares * step;
                c.piece(d + uint32_t(col - n0), row0, split * sh.part_rows + row0, col, factor, ok, next < end ? next : -1,
                        release);
            }
            if (++half == 2) half = 0, half_phase ^= 1;
        }
        if (lane == 0) tc::stores_read();
    }
    __syncwarp();
    tc::fence_before();
    if (kPair)
        tc::cluster_sync();
    else
        __syncthreads();
    if (warp == 1) {
        tc::fence_after();
        tc::tmem_free<kPair>(tmem, L::kColumns);
    }
}

// A few rows of x (a decoding step): one warp per output column, all rows at once, the weights read once and straight
// from memory. Tiles of 128 rows would multiply zeros, and their set-up takes longer than this product. kFewRows rows are
// the most that one pass carries; a second dimension of CTAs carries more.
constexpr int kFewRows = 8;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
few_rows_kernel(const T *__restrict__ x, int64_t x_ld, const T *__restrict__ w, int64_t w_ld, int M, int N, int K,
                const __grid_constant__ Epilogue ep)
{
    using E = Elt<T>;
    const int lane = threadIdx.x & 31, n = blockIdx.x * 8 + (threadIdx.x >> 5), m0 = blockIdx.y * kFewRows;
    if (n >= N) return;
    const int rows = M - m0 < kFewRows ? M - m0 : kFewRows;
    const T *wn = w + int64_t(n) * w_ld, *xm = x + int64_t(m0) * x_ld;
    float sum[kFewRows] = {};
    constexpr int kStep = VEC ? 8 : 1;
#pragma unroll 2
    for (int k = lane * kStep; k < K; k += 32 * kStep) {
        float a[kStep], b[kStep];
        if constexpr (VEC)
            E::unpack(__ldg(reinterpret_cast<const uint4 *>(wn + k)), a);
        else
            a[0] = E::to_acc(__ldg(wn + k));
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
            if (r < rows) {
                if constexpr (VEC)
                    E::unpack(__ldg(reinterpret_cast<const uint4 *>(xm + r * x_ld + k)), b);
                else
                    b[0] = E::to_acc(__ldg(xm + r * x_ld + k));
#pragma unroll
                for (int i = 0; i < kStep; ++i) sum[r] = fmaf(a[i], b[i], sum[r]);
            }
        }
    }
    float mine = 0.0f;  // lane r keeps row r
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], o);
        if (lane == r) mine = sum[r];
    }
    if (lane < rows) {
        const int64_t row = m0 + lane;
        if (ep.bias) mine += E::to_acc(__ldg(static_cast<const T *>(ep.bias) + n));
        const float side = ep.side ? E::to_acc(__ldg(static_cast<const T *>(ep.side) + row * ep.side_ld + n)) : 0.0f;
        mine = finish_as(ep, mine, side);
        static_cast<T *>(ep.out)[row * ep.out_ld + n] = E::from_acc(mine);
        if (ep.low) static_cast<T *>(ep.low)[row * ep.out_ld + n] = low_part<T>(mine);
    }
}
template <typename T>
cudaError_t run_few_rows(const T *x, int64_t x_ld, const T *w, int64_t w_ld, int M, int N, int K, const Epilogue &ep,
                         cudaStream_t s)
{
    const dim3 grid(unsigned((N + 7) / 8), unsigned((M + kFewRows - 1) / kFewRows));
    auto even = [](const void *p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; };
    if (K % 8 == 0 && even(x, x_ld) && even(w, w_ld))
        few_rows_kernel<T, true><<<grid, 256, 0, s>>>(x, x_ld, w, w_ld, M, N, K, ep);
    else
        few_rows_kernel<T, false><<<grid, 256, 0, s>>>(x, x_ld, w, w_ld, M, N, K, ep);
    return cudaGetLastError();
}

// The parts of a split sum, added in their order, and the epilogue.
template <typename T>
__global__ void __launch_bounds__(256)
join_kernel(const float *__restrict__ part, int splits, int64_t part_rows, int64_t M, int N, const Epilogue ep)
{
    const int groups = (N + 7) / 8, ld = groups * 8;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < M * groups; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / groups;
        const int col = int(i % groups) * 8, n = N - col < 8 ? N - col : 8;
        float v[8] = {};
        for (int s = 0; s < splits; ++s) {
            const float4 *p = reinterpret_cast<const float4 *>(part + (s * part_rows + row) * ld + col);
            const float4 a = __ldg(p), b = __ldg(p + 1);
            v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
            v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
        }
        finish_in_place<T>(ep, v, row, col, n);
    }
}

// [rows, cols] of any stride to rows at multiples of 16 bytes.
template <typename T>
__global__ void __launch_bounds__(256) restride_kernel(const T *__restrict__ src, int64_t src_ld, T *__restrict__ dst, int64_t dst_ld,
                                int64_t rows, int cols)
{
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < rows * dst_ld; i += int64_t(gridDim.x) * 256) {
        const int64_t r = i / dst_ld;
        const int c = int(i % dst_ld);
        dst[i] = c < cols ? src[r * src_ld + c] : Elt<T>::from_acc(0.0f);
    }
}

// Column sums (of a matrix, or of one in two parts): each CTA adds up a run of rows of 256 columns in float; the runs' sums
// are added in order afterwards.
constexpr int kSumRows = 8;
template <typename T>
__global__ void __launch_bounds__(256) column_sums_kernel(const T *__restrict__ high,
                                                          const T *__restrict__ low, int64_t ld, int64_t rows, int cols,
                                                          int64_t run, float *__restrict__ part)
{
    using E = Elt<T>;
    __shared__ float sums[kSumRows][256 + 8];
    const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
    const int col = blockIdx.x * 256 + tx * 8;
    float acc[8] = {};
    const int64_t first = int64_t(blockIdx.y) * run, end = first + run < rows ? first + run : rows;
    for (const T *g : {low, high}) {
        if (!g || col >= cols) continue;
        for (int64_t r = first + ty; r < end; r += kSumRows) {
            float v[8];
            if (col + 8 <= cols) {
                E::unpack(__ldg(reinterpret_cast<const uint4 *>(g + r * ld + col)), v);
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = col + c < cols ? E::to_acc(__ldg(g + r * ld + col + c)) : 0.0f;
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) acc[c] += v[c];
        }
        if (g == low) {
#pragma unroll
            for (int c = 0; c < 8; ++c) acc[c] *= 1.0f / kLowScale<T>;
        }
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) sums[ty][tx * 8 + c] = acc[c];
    __syncthreads();
    const int mine = blockIdx.x * 256 + threadIdx.x;
    if (mine < cols) {
        float s = 0.0f;
        for (int y = 0; y < kSumRows; ++y) s += sums[y][threadIdx.x];
        part[int64_t(blockIdx.y) * cols + mine] = s;
    }
}
// Sums of `each` runs at a time.
__global__ void __launch_bounds__(256)
column_fold_kernel(const float *__restrict__ part, int64_t runs, int64_t each, int cols, float *__restrict__ out)
{
    const int c = blockIdx.x * 256 + threadIdx.x;
    const int64_t first = blockIdx.y * each, end = first + each < runs ? first + each : runs;
    if (c >= cols) return;
    float s = 0.0f;
#pragma unroll 8
    for (int64_t i = first; i < end; ++i) s += __ldg(part + i * cols + c);
    out[int64_t(blockIdx.y) * cols + c] = s;
}
// 32 columns a CTA, eight threads each, whose sums are added in order.
template <typename T>
__global__ void __launch_bounds__(256)
column_join_kernel(const float *__restrict__ part, int runs, int cols, T *__restrict__ out)
{
    __shared__ float sums[8][33];
    const int tx = threadIdx.x % 32, ty = threadIdx.x / 32, c = blockIdx.x * 32 + tx;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 4
        for (int i = ty; i < runs; i += 8) s += __ldg(part + int64_t(i) * cols + c);
    }
    sums[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < cols) {
        for (int y = 1; y < 8; ++y) s += sums[y][tx];
        out[c] = Elt<T>::from_acc(s);
    }
}

// --------------------------------------------------------------------------------------------------------- host side

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder()
{
    static const EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) !=
                cudaSuccess || found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// A [rows, cols] matrix in memory, 16-byte rows, copied in boxes of 128 bytes x `box_rows` rows.
template <typename T>
bool make_map(CUtensorMap *map, const void *p, int64_t rows, int64_t cols, int64_t ld, int box_rows)
{
    const EncodeFn encode = encoder();
    if (!encode) return false;
    const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)}, strides[1] = {cuuint64_t(ld) * sizeof(T)};
    const cuuint32_t box[2] = {128 / sizeof(T), cuuint32_t(box_rows)}, one[2] = {1, 1};
    CUtensorMapDataType type = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    if constexpr (sizeof(T) == 2)
        type = Elt<T>::kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return encode(map, type, 2, const_cast<void *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Products of a few rows need no tiles (and no copies for TMA), as long as re-reading the rows of x for every column does
// not take longer than a tile's set-up: 8 rows, us: 1024 x 640 5.0 (tiles 8.4), 1024 x 2048 7.7 (9.8), 4096 x 4096 28 (14).
bool takes_few_rows(int64_t M, int64_t N, int64_t len) { return M <= 16 && N * len <= (int64_t(1) << 22); }

int steps_of(int64_t len) { return int((len + kBK - 1) / kBK); }

// How a product of M x N outputs and a sum of `steps` steps is cut: the width of its tiles and the parts of its sum.
struct Cut {
    int bn, splits, steps_per_split;
    int rows() const { return bn == 256 ? 2 * kBM : kBM; }  // of a tile (of both CTAs of a pair)
    int64_t tiles(int64_t M, int N) const { return ((M + rows() - 1) / rows()) * ((N + bn - 1) / bn); }
    int at_once() const { return bn == 256 ? kNumSMs / 2 : kNumSMs; }
};
Cut cut_product(int64_t M, int N, int steps)
{
    // The width by what its waves of tiles take, in ns: a launch, and for each wave the steps or the epilogue, whichever is
    // longer. Measured with each width forced: 4000 x 512 x 64 (one step) 6.0 / 5.1 / 7.9 us at 64 / 128 / 256,
    // 40009 x 640 x 64 33.6 / 21.3 / 24.8, 40009 x 640 x 512 72 / 42 / 34, 4000 x 1024 x 640 19.4 / 12.7 / 11.5.
    struct Width {
        int bn, launch, step, epilogue;
    };
    constexpr Width widths[] = {{256, 5500, 520, 3100}, {128, 4000, 420, 1600}, {64, 4500, 390, 1350}};
    Cut c{0, 1, steps};
    int64_t best = 0;
    for (const Width &w : widths) {
        if (w.bn > 64 && w.bn / 2 >= N) continue;
        const Cut t{w.bn, 1, steps};
        const int64_t waves = (t.tiles(M, N) + t.at_once() - 1) / t.at_once(), main = int64_t(steps) * w.step;
        const int64_t cost = w.launch + waves * (main > w.epilogue ? main : w.epilogue);
        if (c.bn == 0 || cost < best) c = t, best = cost;
    }
    // split long sums of few tiles (of none where there are no rows), at least eight steps a part
    if (M > 0 && c.tiles(M, N) * 2 <= kNumSMs && steps >= 32) {
        // wide tiles again: parts give the SMs their work
        c.bn = N > 128 && M > 128 ? 256 : (N > 64 ? 128 : 64);
        int64_t parts = c.at_once() / c.tiles(M, N);
        if (parts > steps / 8) parts = steps / 8;
        if (parts < 1) parts = 1;
        c.steps_per_split = int((steps + parts - 1) / parts);
        c.splits = (steps + c.steps_per_split - 1) / c.steps_per_split;
    }
    return c;
}
// Parts are [splits * rows of whole tiles, N up to a multiple of 8] floats.
int64_t part_rows(int64_t M) { return align_up(M, 2 * kBM); }
int64_t part_bytes(int64_t M, int N, const Cut &c)
{
    return c.splits > 1 ? 4 * c.splits * part_rows(M) * align_up(N, 8) : 0;
}

struct Matrix {  // [rows, cols], `mn`: its columns are the output's and its rows the sum's
    const void *p;
    int64_t rows, cols, ld;
    bool mn;
    const void *low = nullptr;  // another matrix of the same shape to be added to it, 2^kLowShift times too large, or none
};

template <typename T, int BN, bool A_MN, bool B_MN>
cudaError_t run_product(const Matrix &a, const Matrix &b, Shape sh, const Epilogue &ep, cudaStream_t s)
{
    using L = Layout<BN>;
    auto kernel = linear_kernel<T, BN, A_MN, B_MN>;
    // The attribute belongs to the device that is current. This comes before the tensor maps: the driver's encoder wants a
    // context bound to the calling thread, which the runtime does with its first call that needs one (a thread of autograd's,
    // or of the caller's, may not have made any).
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::most_bytes());
    if (e != cudaSuccess) return e;
    CUtensorMap ma, mb, mo{}, ms{}, ml{};
    bool good = make_map<T>(&ma, a.p, a.rows, a.cols, a.ld, A_MN ? kBK : kBM) &&
                make_map<T>(&mb, b.p, b.rows, b.cols, b.ld, B_MN ? kBK : L::kRowsB);
    if (ep.mode == kPart)
        good = good && make_map<float>(&mo, ep.out, sh.splits * part_rows(sh.M), sh.N, ep.out_ld, 32);
    else if (ep.tma_out)
        good = good && make_map<T>(&mo, ep.out, sh.M, sh.N, ep.out_ld, 32);
    if (ep.side) good = good && make_map<T>(&ms, ep.side, sh.M, sh.N, ep.side_ld, 32);
    // the low part of A, or of dz on its way out (never both)
    if (a.low) good = good && make_map<T>(&ml, a.low, a.rows, a.cols, a.ld, A_MN ? kBK : kBM);
    if (ep.low) good = good && make_map<T>(&ml, ep.low, sh.M, sh.N, ep.out_ld, 32);
    if (!good) return cudaErrorInvalidValue;
    const int pieces = ep.pieces();
    sh.stages = L::stages(pieces);
    const int ctas = L::kPair ? 2 : 1;
    const int64_t total = sh.tiles_m * sh.tiles_n * sh.splits * ctas;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(total < kNumSMs ? total : kNumSMs));
    cfg.blockDim = dim3(L::kThreads);
    cfg.dynamicSmemBytes = L::bytes(pieces);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = L::kPair ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, ma, mb, mo, ms, ml, sh, ep);
}

template <typename T, bool A_MN, bool B_MN>
cudaError_t run_product_bn(int bn, const Matrix &a, const Matrix &b, const Shape &sh, const Epilogue &ep, cudaStream_t s)
{
    switch (bn) {
    case 256: return run_product<T, 256, A_MN, B_MN>(a, b, sh, ep, s);
    case 128: return run_product<T, 128, A_MN, B_MN>(a, b, sh, ep, s);
    case 64: return run_product<T, 64, A_MN, B_MN>(a, b, sh, ep, s);
    }
    return cudaErrorInvalidValue;
}

// out[M, N] = epilogue(sum over `len` of a * b); `part`: part_bytes() of workspace.
template <typename T>
cudaError_t product(const Matrix &a, const Matrix &b, int64_t M, int N, int64_t len, Epilogue ep, float *part, cudaStream_t s)
{
    if (!a.mn && !b.mn && takes_few_rows(M, N, len))
        return run_few_rows<T>(static_cast<const T *>(a.p), a.ld, static_cast<const T *>(b.p), b.ld, int(M), N, int(len), ep,
                               s);
    const int steps = steps_of(len) * (a.low ? 2 : 1);
    const Cut c = cut_product(M, N, steps);
    Shape sh{};
    sh.M = M, sh.N = N;
    sh.steps = steps;
    sh.half_steps = a.low ? steps / 2 : 0;
    sh.steps_per_split = c.steps_per_split, sh.splits = c.splits;
    sh.tiles_m = (M + c.rows() - 1) / c.rows(), sh.tiles_n = (N + c.bn - 1) / c.bn;
    sh.part_rows = part_rows(M);
    auto on16 = [](const void *p, int64_t ld) {
        return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0);
    };
    ep.tma_out = on16(ep.out, ep.out_ld);
    ep.vec = N % 8 == 0 && ep.tma_out && on16(ep.side, ep.side_ld);
    Epilogue here = ep;
    if (c.splits > 1) {
        here = Epilogue{};
        here.mode = kPart, here.out = part, here.out_ld = align_up(N, 8), here.tma_out = true;
    }
    cudaError_t e;
    if (a.mn)
        e = run_product_bn<T, true, true>(c.bn, a, b, sh, here, s);
    else if (b.mn)
        e = run_product_bn<T, false, true>(c.bn, a, b, sh, here, s);
    else
        e = run_product_bn<T, false, false>(c.bn, a, b, sh, here, s);
    if (e != cudaSuccess || c.splits == 1) return e;
    const int64_t items = M * ((N + 7) / 8), blocks = (items + 255) / 256;
    join_kernel<T><<<unsigned(blocks < kNumSMs * 16 ? blocks : kNumSMs * 16), 256, 0, s>>>(part, c.splits, part_rows(M), M, N, ep);
    return cudaGetLastError();
}

// Workspace: copies of matrices whose rows TMA cannot take, dz, parts of split sums, column sums.
int64_t padded(int64_t cols) { return align_up(cols, 8); }
int64_t copy_bytes(int64_t rows, int64_t cols, int64_t ld)
{
    return ld % 8 ? align_up(rows * padded(cols) * 2, 256) : 0;
}
constexpr int kMostRuns = 256;

// dz is rounded to the operands' type for its two products. Rounded once it would cost their results as much again as
// their own rounding does, so it goes into them as two parts; relu's is exact as it is.
int parts_of(const cwrnnt_linear &p)
{
    return p.activation == CWRNNT_ACT_TANH || p.activation == CWRNNT_ACT_SILU ? 2 : 1;
}

struct LinearPlan {
    int64_t x, w, g, dz, low, side, part, sums, total;  // offsets
};
LinearPlan plan_linear(const cwrnnt_linear &p, bool backward, bool residual)
{
    LinearPlan q{};
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += align_up(bytes, 256);
        return here;
    };
    q.side = take(residual ? copy_bytes(p.n_rows, p.n_out, p.n_out) : 0);
    const bool copies = backward || !takes_few_rows(p.n_rows, p.n_out, p.n_in);
    q.x = take(copies ? copy_bytes(p.n_rows, p.n_in, p.x_stride) : 0);
    q.w = take(copies ? copy_bytes(p.n_out, p.n_in, p.w_stride) : 0);
    auto most = [](int64_t a, int64_t b) { return a > b ? a : b; };
    int64_t parts = 0;
    if (!backward || p.activation != CWRNNT_ACT_NONE)
        parts = part_bytes(p.n_rows, p.n_out, cut_product(p.n_rows, p.n_out, steps_of(p.n_in)));
    if (backward) {
        q.g = take(copy_bytes(p.n_rows, p.n_out, p.g_stride));
        if (p.activation != CWRNNT_ACT_NONE) q.dz = take(p.n_rows * padded(p.n_out) * 2);
        if (parts_of(p) == 2) q.low = take(p.n_rows * padded(p.n_out) * 2);
        parts = most(parts, part_bytes(p.n_rows, p.n_in, cut_product(p.n_rows, p.n_in, steps_of(p.n_out) * parts_of(p))));
        parts = most(parts, part_bytes(p.n_out, p.n_in, cut_product(p.n_out, p.n_in, steps_of(p.n_rows) * parts_of(p))));
        q.sums = take(4 * (kMostRuns + (p.n_rows + 31) / 32) * int64_t(p.n_out));
    }
    q.part = take(parts);
    q.total = at > 0 ? at : 256;
    return q;
}

template <typename T>
cudaError_t restride(const void *src, int64_t ld, int64_t rows, int64_t cols, void *dst, cudaStream_t s)
{
    const int64_t items = rows * padded(cols), blocks = (items + 255) / 256;
    if (items == 0) return cudaSuccess;
    restride_kernel<T><<<unsigned(blocks < kNumSMs * 32 ? blocks : kNumSMs * 32), 256, 0, s>>>(
        static_cast<const T *>(src), ld, static_cast<T *>(dst), padded(cols), rows, int(cols));
    return cudaGetLastError();
}

// `m` as TMA can take it, copied to `room` if need be.
template <typename T>
cudaError_t readable(Matrix &m, char *room, cudaStream_t s)
{
    if (m.ld % 8 == 0) return cudaSuccess;
    const cudaError_t e = restride<T>(m.p, m.ld, m.rows, m.cols, room, s);
    m.p = room, m.ld = padded(m.cols);
    return e;
}

#define CWRNNT_TRY(call)                                   \
    do {                                                   \
        const cudaError_t e_ = (call);                     \
        if (e_ != cudaSuccess) return e_;                  \
    } while (0)

template <typename T>
cudaError_t linear_forward(const cwrnnt_linear &p, const void *x, const void *w, const void *bias, const void *residual,
                           char *ws, void *y, cudaStream_t s)
{
    const LinearPlan q = plan_linear(p, false, residual != nullptr);
    Matrix a{x, p.n_rows, p.n_in, p.x_stride, false}, b{w, p.n_out, p.n_in, p.w_stride, false};
    if (!takes_few_rows(p.n_rows, p.n_out, p.n_in)) {
        CWRNNT_TRY(readable<T>(a, ws + q.x, s));
        CWRNNT_TRY(readable<T>(b, ws + q.w, s));
    }
    Epilogue ep{};
    ep.mode = kStore, ep.act = p.activation, ep.bias = bias;
    Matrix r{residual, p.n_rows, p.n_out, p.n_out, false};
    if (residual && !takes_few_rows(p.n_rows, p.n_out, p.n_in)) CWRNNT_TRY(readable<T>(r, ws + q.side, s));
    ep.side = r.p, ep.side_ld = r.ld;
    ep.out = y, ep.out_ld = p.n_out;
    return product<T>(a, b, p.n_rows, p.n_out, p.n_in, ep, reinterpret_cast<float *>(ws + q.part), s);
}

template <typename T>
cudaError_t linear_backward(const cwrnnt_linear &p, const void *x, const void *w, const void *bias, const void *g,
                            char *ws, void *grad_x, void *grad_w, void *grad_b, cudaStream_t s)
{
    const LinearPlan q = plan_linear(p, true, false);
    float *part = reinterpret_cast<float *>(ws + q.part);
    Matrix mx{x, p.n_rows, p.n_in, p.x_stride, false}, mw{w, p.n_out, p.n_in, p.w_stride, false};
    Matrix dz{g, p.n_rows, p.n_out, p.g_stride, false};
    const bool act = p.activation != CWRNNT_ACT_NONE;
    if (act || grad_w) CWRNNT_TRY(readable<T>(mx, ws + q.x, s));
    if (act || grad_x) CWRNNT_TRY(readable<T>(mw, ws + q.w, s));
    // column sums: of the epilogue's pieces of 32 rows where it forms dz, else of runs of rows of the matrix
    float *sums = reinterpret_cast<float *>(ws + q.sums), *folded = sums + (p.n_rows + 31) / 32 * int64_t(p.n_out);
    int64_t runs = 0;
    CWRNNT_TRY(readable<T>(dz, ws + q.g, s));
    if (act) {
        Epilogue ep{};
        ep.mode = kSlope, ep.act = p.activation, ep.bias = bias;
        ep.side = dz.p, ep.side_ld = dz.ld;
        ep.out = ws + q.dz, ep.out_ld = padded(p.n_out);
        const bool tiles = !takes_few_rows(p.n_rows, p.n_out, p.n_in) &&
                           cut_product(p.n_rows, p.n_out, steps_of(p.n_in)).splits == 1;
        if (tiles && grad_b) ep.sums = sums, runs = (p.n_rows + 31) / 32;
        ep.low = parts_of(p) == 2 ? ws + q.low : nullptr;
        CWRNNT_TRY(product<T>(mx, mw, p.n_rows, p.n_out, p.n_in, ep, part, s));
        dz.p = ws + q.dz, dz.ld = padded(p.n_out);
        dz.low = ep.low;
    }
    if (grad_b) {
        const int64_t across = (p.n_out + 255) / 256;
        if (runs == 0) {
            // enough runs to fill the GPU with CTAs of 256 columns
            runs = (kNumSMs * 4 + across - 1) / across;
            const int64_t most = (p.n_rows + 63) / 64;
            if (runs > most) runs = most;
            if (runs > kMostRuns) runs = kMostRuns;
            const int64_t run = (p.n_rows + runs - 1) / runs;
            column_sums_kernel<T><<<dim3(unsigned(across), unsigned(runs)), 256, 0, s>>>(
                static_cast<const T *>(dz.p), static_cast<const T *>(dz.low), dz.ld, p.n_rows, p.n_out, run, sums);
            CWRNNT_TRY(cudaGetLastError());
        }
        if (runs > kMostRuns) {
            const int64_t each = (runs + kMostRuns / 2 - 1) / (kMostRuns / 2), groups = (runs + each - 1) / each;
            column_fold_kernel<<<dim3(unsigned(across), unsigned(groups)), 256, 0, s>>>(sums, runs, each, p.n_out, folded);
            CWRNNT_TRY(cudaGetLastError());
            sums = folded, runs = groups;
        }
        column_join_kernel<T><<<unsigned((p.n_out + 31) / 32), 256, 0, s>>>(sums, int(runs), p.n_out,
                                                                              static_cast<T *>(grad_b));
        CWRNNT_TRY(cudaGetLastError());
    }
    if (grad_x) {
        Epilogue ep{};
        ep.out = grad_x, ep.out_ld = p.n_in;
        Matrix b = mw;
        b.mn = true;
        CWRNNT_TRY(product<T>(dz, b, p.n_rows, p.n_in, p.n_out, ep, part, s));
    }
    if (grad_w) {
        Epilogue ep{};
        ep.out = grad_w, ep.out_ld = p.n_in;
        Matrix a = dz, b = mx;
        a.mn = b.mn = true;
        CWRNNT_TRY(product<T>(a, b, p.n_out, p.n_in, p.n_rows, ep, part, s));
    }
    return cudaSuccess;
}

}  // namespace

int64_t linear_workspace(const cwrnnt_linear &p, bool backward, bool residual)
{
    return plan_linear(p, backward, residual).total;
}

cudaError_t launch_linear(const cwrnnt_linear &p, const void *x, const void *w, const void *bias, const void *residual,
                          void *workspace, void *y, cudaStream_t s)
{
    if (p.dtype == CWRNNT_F16)
        return linear_forward<__half>(p, x, w, bias, residual, static_cast<char *>(workspace), y, s);
    return linear_forward<__nv_bfloat16>(p, x, w, bias, residual, static_cast<char *>(workspace), y, s);
}

cudaError_t launch_linear_grad(const cwrnnt_linear &p, const void *x, const void *w, const void *bias, const void *g,
                               void *workspace, void *grad_x, void *grad_w, void *grad_b, cudaStream_t s)
{
    char *ws = static_cast<char *>(workspace);
    if (p.dtype == CWRNNT_F16) return linear_backward<__half>(p, x, w, bias, g, ws, grad_x, grad_w, grad_b, s);
    return linear_backward<__nv_bfloat16>(p, x, w, bias, g, ws, grad_x, grad_w, grad_b, s);
}

}  // namespace cwrnnt
