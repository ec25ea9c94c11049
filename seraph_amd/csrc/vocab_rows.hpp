// vocab_rows.hpp - what the objectives over vocabulary logits share: which rows are supervised, how a row is
// addressed, reductions over a workgroup, and the exponentials.
//
// All of them are a softmax over rows of `cols` logits and, for the gradient, one value per logit that follows from
// the logit and a few numbers of its row.  At six to ten operations per eight bytes every kernel here is bound by
// memory; what differs between them is how often a logit crosses it.
#pragma once

#include <math.h>

#include "common.hpp"

namespace seraph {

constexpr float kLowest = -3.402823466e38f;       // the type's lowest value: a maximum over nothing, or over masked logits

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4a4 __attribute__((ext_vector_type(4), aligned(4)));      // 16 bytes on a 4-byte boundary

// What a row needs besides its maximum m and its sum of exp((z - m) / T):
enum Extra {
    kNone,        // nothing
    kEntropy,     // the sum of exp(z - m) (z - m)      (T = 1)
    kSecond,      // the sum of exp(z - m), beside the one at T
    kSquare       // the same at T = 2, where it is the square of the first
};
// Whether the gradient follows from the exponential alone, which then takes the logit's register; else it is formed again
// from the logit, rather than kept beside it.
constexpr bool holds_exp(int extra) { return extra == kNone || extra == kSquare; }

struct RowStats { float m, s, x; };

// The factor log2(e) / T in two parts.  Its FP32 rounding alone (1.3e-8 of it at T = 1) shifts every argument the same way,
// which the logarithm of a sum keeps: 1.3e-8 times the mean of m - z under the softmax, 7e-8 a token where that is 5.5, and
// a sequence's score adds its tokens up.  With both parts the errors of such tokens measured 1e-9 to 5e-9 in the mean, 4e-8 to
// 9e-8 rms.
struct ExpScale {
    float hi, lo;
    static ExpScale of(double inv_temp) {
        const double k = 1.4426950408889634074 * inv_temp;
        float hi = (float)k;
        if ((double)hi >= k) hi = nextafterf(hi, 0.0f);           // both parts positive: -inf times them adds up to -inf
        return ExpScale{hi, (float)(k - (double)hi)};
    }
};
constexpr ExpScale kUnitScale{1.442695021629333f, 1.92596298909109e-8f};      // ExpScale::of(1)

// exp((z - m) / T).  The difference is formed first: m k could overflow where every logit of a row is the type's
// lowest value, and (z - m) k keeps the bits that fma(z, k, -m k) would lose for a large m.
__device__ __forceinline__ float exp_of(float z, float m, ExpScale k) {
    const float d = z - m;
    return __builtin_amdgcn_exp2f(fmaf(d, k.hi, d * k.lo));
}

// The same for the gradient, where nothing adds up over tokens: the first part of the factor alone.
__device__ __forceinline__ float exp_once(float z, float m, ExpScale k) { return __builtin_amdgcn_exp2f((z - m) * k.hi); }

// log s in 64 bits, off by 1e-7 at most: the exponent is exact, the logarithm of the mantissa lies in [-ln 2, 0].  A few
// instructions and registers, where log(double) needs dozens of both beside a row that fills a lane's registers.
__device__ __forceinline__ double log_of(float s) {
    return (double)__builtin_amdgcn_frexp_expf(s) * 0.693147180559945309 + (double)(__builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(s)) * 0.6931471805599453f);
}

// log of a row's sum in 64 bits, for log-probabilities that are added up over tokens.  The hardware's 2^x is low by 3.4e-9 of its
// value in the mean (over fractions of its argument 2.3e-9 to 4.3e-9; 4 million arguments in (-24, 0), rms 2.7e-8), and exact at 0: the
// row's largest term is 1 or a few times that, the others get what they lack on average.
__device__ __forceinline__ double log_of_sum(float s) { return log((double)s + 3.4e-9 * fmax((double)s - 1.0, 0.0)); }

// e^d of a 64-bit d to one or two units of its last place: d in two floats, and 2^n times the exponential of a fraction that FP32
// holds to 2^-25.  (exp_of rounds its argument to FP32, which costs |d| / 2 units.)
__device__ __forceinline__ float exp_of_wide(double d) {
    const float hi = (float)d, t = hi * kUnitScale.hi, n = rintf(t), lo = (float)(d - (double)hi);
    const float e = ldexpf(__builtin_amdgcn_exp2f(fmaf(hi, kUnitScale.hi, -n) + fmaf(hi, kUnitScale.lo, lo * kUnitScale.hi)), (int)n);
    return fabsf(t) < 200.0f ? e : t < 0.0f ? 0.0f : t > 0.0f ? INFINITY : t;
}

// e^d - 1 (rise) and e^d - 1 - d (excess), each to a few units of its last place.  Near zero, where the differences would cancel, the
// excess by its series and the rise as excess + d; from |d| = 1 on both from e^d itself: there the excess would lose the 1
// beside a large |d|, and it is infinite at d = -inf, where the rise is -1.  Without branches: one lane computes it
// while its workgroup waits, and a branch around e^d took 0.07 us of the 21 that the policy loss takes at 2048 x 8192.
struct ExpLess { float rise, excess; };
__device__ __forceinline__ ExpLess exp_less(double d) {
    const float x = (float)d;
    float p = 1.0f / 3628800.0f;                                  // x^2 (1/2! + x/3! + ... + x^8/10!)
    p = fmaf(p, x, 1.0f / 362880.0f);
    p = fmaf(p, x, 1.0f / 40320.0f);
    p = fmaf(p, x, 1.0f / 5040.0f);
    p = fmaf(p, x, 1.0f / 720.0f);
    p = fmaf(p, x, 1.0f / 120.0f);
    p = fmaf(p, x, 1.0f / 24.0f);
    p = fmaf(p, x, 1.0f / 6.0f);
    p = fmaf(p, x, 0.5f);
    const bool near = fabs(d) < 1.0;
    const float series = x * x * p;
    const double rise = (double)exp_of_wide(d) - 1.0;
    return ExpLess{near ? series + x : (float)rise, near ? series : (float)(rise - d)};
}

// e^d, d <= 0, to 1e-11 of it: where results of parts of a row are joined.  The hardware's 2^x is low by 3.4e-9 in the mean; a
// row's logarithm keeps that once for every factor between a logit and the row's sum, and a score adds it up over its tokens.
__device__ __forceinline__ double exp_below(double d) {
    if (!(d > -200.0)) return d != d ? d : 0.0;
    const double t = d * 1.4426950408889634074, n = rint(t), x = (t - n) * 0.693147180559945309;
    double p = 1.0 / 362880.0;                                    // 1 + x + ... + x^9/9!, |x| <= log(2)/2
    p = fma(p, x, 1.0 / 40320.0);
    p = fma(p, x, 1.0 / 5040.0);
    p = fma(p, x, 1.0 / 720.0);
    p = fma(p, x, 1.0 / 120.0);
    p = fma(p, x, 1.0 / 24.0);
    p = fma(p, x, 1.0 / 6.0);
    p = fma(p, x, 0.5);
    p = fma(p, x, 1.0);
    return ldexp(fma(p, x, 1.0), (int)n);
}

template <int EXTRA>
__device__ __forceinline__ float extra_of(float z, float m, float e) {
    if (EXTRA == kEntropy) return e > 0.0f ? e * (z - m) : (e == 0.0f ? 0.0f : e);      // exp(-inf) (-inf) counts 0, NaN stays
    if (EXTRA == kSecond) return exp_of(z, m, kUnitScale);
    if (EXTRA == kSquare) return e * e;
    return 0.0f;
}

// Reductions over a wave by data-parallel moves: lanes 1, 2, 4 and 8 below within each row of 16, then the rows' last
// lanes into the next rows; lane 63 ends with the whole and hands it to all as a scalar.  Six dependent additions, where
// shuffles through the LDS crossbar put some 60 cycles behind each.
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float v, float otherwise) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, otherwise), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v, double otherwise) {
    const uint64_t a = __builtin_bit_cast(uint64_t, v), b = __builtin_bit_cast(uint64_t, otherwise);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)b, (int)(uint32_t)a, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)(b >> 32), (int)(uint32_t)(a >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ float last_lane(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63)); }
__device__ __forceinline__ double last_lane(double v) {
    const uint64_t a = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)a, 63), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(a >> 32), 63);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
enum { kShr1 = 0x111, kShr2 = 0x112, kShr4 = 0x114, kShr8 = 0x118, kBcast15 = 0x142, kBcast31 = 0x143 };
template <class T>
__device__ __forceinline__ T wave_total(T v) {                    // every lane of the wave is active
    v += moved<kShr1, 0xf>(v, (T)0);
    v += moved<kShr2, 0xf>(v, (T)0);
    v += moved<kShr4, 0xf>(v, (T)0);
    v += moved<kShr8, 0xf>(v, (T)0);
    v += moved<kBcast15, 0xa>(v, (T)0);
    v += moved<kBcast31, 0xc>(v, (T)0);
    return last_lane(v);
}
__device__ __forceinline__ float wave_top(float v) {
    v = fmaxf(v, moved<kShr1, 0xf>(v, v));
    v = fmaxf(v, moved<kShr2, 0xf>(v, v));
    v = fmaxf(v, moved<kShr4, 0xf>(v, v));
    v = fmaxf(v, moved<kShr8, 0xf>(v, v));
    v = fmaxf(v, moved<kBcast15, 0xa>(v, v));
    v = fmaxf(v, moved<kBcast31, 0xc>(v, v));
    return last_lane(v);
}

template <int BLOCK>
__device__ __forceinline__ float block_max(float v, float* lds) {
    v = wave_top(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = lds[0];
#pragma unroll
    for (int w = 1; w < BLOCK / 64; w++) r = fmaxf(r, lds[w]);
    return r;
}
template <int BLOCK, class T>
__device__ __forceinline__ T block_sum(T v, T* lds) {
    v = wave_total(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    T r = lds[0];
#pragma unroll
    for (int w = 1; w < BLOCK / 64; w++) r += lds[w];
    return r;
}
// both sums over the workgroup behind one barrier; lds holds 2 BLOCK / 64 floats
template <int BLOCK>
__device__ __forceinline__ void block_sum2(float& a, float& b, float* lds) {
    a = wave_total(a);
    b = wave_total(b);
    if ((threadIdx.x & 63) == 0) {
        lds[threadIdx.x >> 6] = a;
        lds[BLOCK / 64 + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = lds[0];
    b = lds[BLOCK / 64];
#pragma unroll
    for (int w = 1; w < BLOCK / 64; w++) { a += lds[w]; b += lds[BLOCK / 64 + w]; }
}

// A row of floats that need not start on a boundary of memory's lines nor hold a multiple of four: `head` single values up to
// the first boundary of 128 bytes, n4 vectors, `tail` single values.  Lanes 0 to 31 of one workgroup hold the head,
// lanes 32 to 34 the tail.  (Vectors from the first 16-byte boundary on would do, but a workgroup's 4 KB would then end
// inside a line, which two of them write a part of: 1000 x 151937 took 9 % longer than 1000 x 151936.)
struct RowShape {
    int head, n4, tail;
    __device__ __forceinline__ RowShape(const float* row, int64_t cols) {
        const int to_boundary = (int)((32u - ((unsigned)(reinterpret_cast<uintptr_t>(row) >> 2) & 31u)) & 31u);
        head = to_boundary < cols ? to_boundary : (int)cols;
        n4 = (int)((cols - head) >> 2);
        tail = (int)((cols - head) & 3);
    }
    // the column of this lane's single value, -1 where it has none
    __device__ __forceinline__ int64_t single(int lane) const {
        if (lane < head) return lane;
        if (lane >= 32 && lane < 32 + tail) return (int64_t)head + (int64_t)n4 * 4 + (lane - 32);
        return -1;
    }
};

// The vectors of a row as a buffer of n4 16-byte slots: a scalar descriptor and one 32-bit offset per lane.  A load past the
// last slot returns zeros and a store past it is dropped, so a slot needs no branch.  The offset is the lane's alone (no scalar
// offset), which is what the range check compares; the address itself may be any multiple of four.
constexpr int kNontemporal = 2;
struct SlotBuffer {
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ SlotBuffer(const float* first, int n4) {
        const uint64_t o = reinterpret_cast<uint64_t>(first);
        const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)o), hi = __builtin_amdgcn_readfirstlane((uint32_t)(o >> 32));
        rsrc = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0, __builtin_amdgcn_readfirstlane(n4 * 16), 0x00020000);
    }
    template <int AUX>
    __device__ __forceinline__ f4 load(int offset) const {
        return __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, offset, 0, AUX));
    }
    template <int AUX>
    __device__ __forceinline__ void store(f4 v, int offset) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(__attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned, v), rsrc, offset, 0, AUX);
    }
};

// Which rows are supervised.
struct Supervision {
    const uint32_t* targets;       // NULL: the op has rows without targets
    const float* weights;          // NULL: all 1
    const uint32_t* seq_starts;    // NULL: one sequence, whose last row counts like the others
    int batch;
    int64_t cols;
    __device__ __forceinline__ bool in_sequence(int64_t row) const {
        if (!seq_starts) return true;
        const int sq = find_seq(seq_starts, batch, row);
        return sq < batch && row >= (int64_t)seq_starts[sq] && row + 1 < (int64_t)seq_starts[sq + 1];
    }
    // (Where a whole workgroup asks for one row these are scalar loads, which do not queue behind the rows' vector loads: a
    // search by all lanes at once, with one vector load instead of a scalar one per step, took 2 us longer of 22.)
    __device__ __forceinline__ bool live(int64_t row) const {
        const uint32_t t = targets ? targets[row] : 0u;
        const float w = weights ? weights[row] : 1.0f;
        return (int)in_sequence(row) & (int)((int64_t)t < cols) & (int)(w != 0.0f);
    }
};

}  // namespace seraph
