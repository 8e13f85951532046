// The AdamW step over many tensors, with moments in 32 bits or in 8 (cx_adamw_step), and the way between
// the 8-bit moments and their values (cx_adamw_states, cx_adamw_set_states).  Formulas and formats:
// include/comprex_gfx950.h.
//
// No product or sum below is contracted: the moments have the same bits whatever the compiler does
// around them, so an 8-bit code never depends on the build.  Where a fused multiply-add is wanted it is
// written out.
#include "cx_tensors.hpp"

#include <cmath>

#pragma clang fp contract(off)

namespace cx {

namespace {

constexpr int kBlock = 256;   // 4 or 8 elements a lane: a fine or a wide piece

// What depends on the step's count.
struct AdamwRates {
    float step;        // lr / (1 - beta1^t)
    float decay;       // lr * weight_decay
    float v_unit;      // 1 / sqrt(1 - beta2^t)
    unsigned long long noise;  // key of the step's rounding, where that is stochastic
};

struct AdamwArgs {
    float beta1, rest1, beta2, rest2, eps, scale;   // rest = 1 - beta, rounded from 64 bits
    AdamwRates rates;
    const AdamwRates* device_rates;                 // replaces `rates` where the count lives on the device
    const float* coefs;
    int per_tensor;
    const int* skip;
    float* moves;                                   // where the moves go, if not into the weights
};

// Mixes 64 bits: the output function of SplitMix64 (Steele, Lea, Flood, "Fast splittable pseudorandom number
// generators", 2014).
constexpr unsigned long long kGolden = 0x9E3779B97F4A7C15ull;
__host__ __device__ inline unsigned long long mixed(unsigned long long z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

__host__ __device__ inline AdamwRates rates_of(double lr, double beta1, double beta2, double weight_decay, long long step,
                                               unsigned long long seed) {
    AdamwRates r;
    const double t = (double)step;
    r.noise = mixed(seed + (unsigned long long)step * kGolden);
    r.step = (float)(lr / (1.0 - pow(beta1, t)));
    r.decay = (float)(lr * weight_decay);
    r.v_unit = (float)(1.0 / sqrt(1.0 - pow(beta2, t)));
    return r;
}

// The step's count on the device: one thread advances it and leaves the rates for the step's kernel.
__global__ void rates_kernel(int* count, long long step, const float* d_lr, double lr, double beta1, double beta2,
                             double weight_decay, unsigned long long seed, const int* skip, AdamwRates* rates) {
    if (skip && *skip) return;
    if (count) step = ++*count;
    *rates = rates_of(d_lr ? (double)*d_lr : lr, beta1, beta2, weight_decay, step, seed);
}

// The moments; g already has its factor.
template <int N>
__device__ __forceinline__ void moments(Vec<float, N> g, const AdamwArgs& a, Vec<float, N>& m, Vec<float, N>& v) {
    m = m * a.beta1 + g * a.rest1;
    v = v * a.beta2 + g * g * a.rest2;
}

// EXACT: square root and quotient correctly rounded.  With moments in 32 bits HBM is the bound either way (25.6 M fp32
// weights 115.4 us, the hardware's root and reciprocal 115.5; 100 M bf16 weights with masters 454 and 460).  With moments
// in 8 bits the instructions nearly are, and root and reciprocal are the hardware's, to one unit in the last place.
template <int N, bool EXACT>
__device__ __forceinline__ Vec<float, N> moves_of(Vec<float, N> m, Vec<float, N> v, const AdamwArgs& a, const AdamwRates& r) {
    Vec<float, N> x;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float below = __builtin_fmaf(EXACT ? __builtin_sqrtf(v[k]) : __builtin_amdgcn_sqrtf(v[k]), r.v_unit, a.eps);
        x[k] = r.step * (EXACT ? m[k] / below : m[k] * __builtin_amdgcn_rcpf(below));
    }
    return x;
}

template <int N> __device__ __forceinline__ Vec<float, N> moved(Vec<float, N> w, Vec<float, N> move, float decay) {
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] -= __builtin_fmaf(decay, w[k], move[k]);
    return w;
}

enum { kWeights = 0, kMasters = 1, kMoves = 2 };   // where a step's moves go

// One piece a workgroup, four elements a lane: everything is asked for before anything is used.
template <typename P, typename G, int TO>
__global__ __launch_bounds__(kBlock) void adamw32_kernel(Pieces ps, GradArgs ga, AdamwArgs a) {
    const Piece c = piece_of<kFine>(ps);
    const G* g = grad_of<G>(c, ga);
    const bool skip = a.skip && *a.skip;
    if (!g || (TO != kMoves && skip)) return;
    const AdamwRates r = a.device_rates ? *a.device_rates : a.rates;
    const float f = factor_of(c, a.coefs, a.per_tensor, a.scale);
    P* p = static_cast<P*>(c.t.param) + c.at;
    float *pm = static_cast<float*>(c.t.m) + c.at, *pv = static_cast<float*>(c.t.v) + c.at;
    float* pw = TO == kMoves ? a.moves + c.t.flat + c.at : c.t.master + c.at;
    const int i = threadIdx.x * 4, k = c.n - i;
    if (k <= 0) return;
    by_length<kBlock * 4>(c, [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        if constexpr (TO == kMoves)
            if (skip) return store_some<4, FULL>(pw + i, Vec<float, 4>{}, k);
        const Vec<G, 4> gx = load_some<4, FULL>(g + i, k);
        Vec<float, 4> m = load_some<4, FULL>(pm + i, k), v = load_some<4, FULL>(pv + i, k), w;
        if constexpr (TO == kMasters) w = load_some<4, FULL>(pw + i, k);
        if constexpr (TO == kWeights) w = to_float<4>(load_some<4, FULL>(p + i, k));
        moments<4>(to_float<4>(gx) * f, a, m, v);
        const Vec<float, 4> move = moves_of<4, true>(m, v, a, r);
        store_some<4, FULL>(pm + i, m, k);
        store_some<4, FULL>(pv + i, v, k);
        if constexpr (TO == kMoves) return store_some<4, FULL>(pw + i, move, k);
        w = moved<4>(w, move, r.decay);
        if constexpr (TO == kMasters) store_some<4, FULL>(pw + i, w, k);
        store_some<4, FULL>(p + i, from_float<P, 4>(w), k);
    });
}

// The other half of a step whose moves went through the exchange.
template <typename P, bool MASTER>
__global__ __launch_bounds__(kBlock) void apply_kernel(Pieces ps, const float* __restrict__ moves, float scale, float decay,
                                                       const float* __restrict__ lr, float weight_decay) {
    const Piece c = piece_of<kFine>(ps);
    if (lr) decay = *lr * weight_decay;
    P* p = static_cast<P*>(c.t.param) + c.at;
    float* pw = c.t.master + c.at;
    const int i = threadIdx.x * 4, k = c.n - i;
    if (k <= 0) return;
    by_length<kBlock * 4>(c, [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        const Vec<float, 4> move = load_some<4, FULL>(moves + c.t.flat + c.at + i, k);
        Vec<float, 4> w;
        if constexpr (MASTER) w = load_some<4, FULL>(pw + i, k);
        else w = to_float<4>(load_some<4, FULL>(p + i, k));
        w = moved<4>(w, move * scale, decay);
        if constexpr (MASTER) store_some<4, FULL>(pw + i, w, k);
        store_some<4, FULL>(p + i, from_float<P, 4>(w), k);
    });
}

// ---- 8-bit moments ---------------------------------------------------------------------------
// Half a wave holds a block of 256 elements, eight a lane.  Four a lane, a block per wave, took 190 us where this takes
// 158 (100 M bf16 weights): twice the waves, each with its way to its piece, its maxima and its quotients.
// A lane's eight are neighbours where weights and gradients have 16 bits (16 bytes a load); where one of them has
// 32 they are two fours, 128 elements apart, so that every load of the wave still covers whole stretches of 512
// bytes (fp32, 25.6 M weights: neighbours 84 us, fours 68 us).
template <bool SPLIT, bool FULL> struct Eight {
    int at, other, n;    // first elements of the two fours within the piece; the piece's length
    __device__ __forceinline__ explicit Eight(int length) : n(length) {
        const int lane = threadIdx.x & 31;
        at = (threadIdx.x >> 5) * CX_STATE_BLOCK + (SPLIT ? lane * 4 : lane * 8);
        other = at + (SPLIT ? 128 : 4);
    }
    template <typename E> __device__ __forceinline__ Vec<E, 8> load(const E* p) const {
        if constexpr (SPLIT) {
            const Vec<E, 4> a = load_some<4, FULL>(p + at, n - at), b = load_some<4, FULL>(p + other, n - other);
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return load_some<8, FULL>(p + at, n - at);
        }
    }
    template <typename E> __device__ __forceinline__ void store(E* p, Vec<E, 8> x) const {
        if constexpr (SPLIT) {
            store_some<4, FULL>(p + at, __builtin_shufflevector(x, x, 0, 1, 2, 3), n - at);
            store_some<4, FULL>(p + other, __builtin_shufflevector(x, x, 4, 5, 6, 7), n - other);
        } else {
            store_some<8, FULL>(p + at, x, n - at);
        }
    }
};

constexpr float kTiny = 0x1p-100f;               // a block below is stored as zeros
constexpr float kVUnit = 0x1.ep-96f;             // V lies here before its bits are cut: exponent field 31, fraction 7/8
constexpr float kVBack = (float)(0x1p96 / 1.875);

// Rounded to nearest, a moment loses every change below half a code step, 3 to 6 % of it, for good: with beta2 = 0.999
// a second moment moves by 0.1 % a step, and falls or rises with its block's largest only.  Rounded stochastically, up
// with the probability that the remainder has of a code step, it follows in expectation: its relative variance settles
// near (code step) * (change a step) / (2 * 0.001) = 0.09 * 0.001 / 0.002, about 0.05.  The remainder is what lies below
// the code's bits in the scaled fp32 value, 20 bits; 16 random bits are added to its upper 16, and half of their unit, so that
// a value that roundings moved off its code by a few units in the last place stays on it.
//
// A wave's random words: a mix of the step's key and the wave's place in the set, the same for all lanes (scalar
// instructions); one more mix for each lane; from there eight words, one for each element, each a bijection of the one
// before, so that every element's is as evenly spread over the steps as the lane's.  Lower half for m, upper for v.
// 100 M bf16 weights take 180 to 195 us with noise and 160 to nearest (six more with three shifts a word): instructions
// are the bound there.  25.6 M in fp32 take 69 us either way.
struct Nearest {};
struct Noise {
    unsigned x[8];
    __device__ __forceinline__ Noise(unsigned long long key, long long place) {
        const unsigned long long z = mixed(key + (unsigned long long)place * kGolden);
        unsigned s = (unsigned)z + (threadIdx.x & 63) * (unsigned)(kGolden >> 32);
        s = (s ^ (s >> 16)) * ((unsigned)(z >> 32) | 1u);
        s = (s ^ (s >> 15)) * 0x4C957F2Du;  // (the lower half of Knuth's multiplier for 64-bit congruences)
        s ^= s >> 16;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            s += s << 9;
            s ^= s >> 14;
            x[k] = s;
        }
    }
    __device__ __forceinline__ unsigned lower(int k) const { return ((x[k] << 4) & 0xffff0u) | 8u; }
    __device__ __forceinline__ unsigned upper(int k) const { return ((x[k] >> 12) & 0xffff0u) | 8u; }
};

struct Codes { unsigned x[2]; };                 // eight of them
using Bytes = Vec<unsigned char, 8>;

// Two maxima over each half of the wave, left in its last lane: four rotations within rows of 16 lanes, then
// every other row takes the row before it along.
__device__ __forceinline__ void half_max(unsigned& a, unsigned& b) {
#define CX_STEP(ctrl, rows)                                                                   \
    {                                                                                         \
        const unsigned x = (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, ctrl, rows, 0xf, false); \
        const unsigned y = (unsigned)__builtin_amdgcn_update_dpp(0, (int)b, ctrl, rows, 0xf, false); \
        a = max(a, x);                                                                        \
        b = max(b, y);                                                                        \
    }
    CX_STEP(0x128, 0xf)  // row_ror:8
    CX_STEP(0x124, 0xf)
    CX_STEP(0x122, 0xf)
    CX_STEP(0x121, 0xf)
    CX_STEP(0x142, 0xa)  // row_bcast:15 into rows 1 and 3
#undef CX_STEP
}

// The largest magnitude among a lane's values; NaN only where there is nothing else.
__device__ __forceinline__ unsigned lane_max(Vec<float, 8> x) {
    float t = __builtin_fabsf(x[0]);
#pragma unroll
    for (int k = 1; k < 8; ++k) t = __builtin_fmaxf(t, __builtin_fabsf(x[k]));
    return __float_as_uint(t);
}
// ... among the finite ones
__device__ __forceinline__ unsigned lane_max_finite(Vec<float, 8> x) {
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const unsigned u = __float_as_uint(x[k]) & 0x7fffffffu;
        top = max(top, u < 0x7f800000u ? u : 0u);
    }
    return top;
}

__device__ __forceinline__ Vec<float, 8> m_value(Codes c, float scale) {
    Vec<float, 8> x;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x[j], true);
        x[4 * j] = lo[0];
        x[4 * j + 1] = lo[1];
        x[4 * j + 2] = hi[0];
        x[4 * j + 3] = hi[1];
    }
    return x * scale;
}
__device__ __forceinline__ Vec<float, 8> v_value(Codes c, float scale) {
    Vec<float, 8> x;
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(((c.x[k / 4] >> (8 * (k % 4))) & 255u) << 20);
    return x * kVBack * scale;
}
__device__ __forceinline__ Codes m_codes(Vec<float, 8> m, float inverse, Nearest) {
    m = m * inverse;
    Codes c;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int u = __builtin_amdgcn_cvt_pk_fp8_f32(m[4 * j], m[4 * j + 1], 0, false);
        c.x[j] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(m[4 * j + 2], m[4 * j + 3], u, true);
    }
    return c;
}
// e4m3's exponent and fraction bits are those of the value after a scaling that puts its smallest normal number at
// fp32's; code 126 is the largest, 127 what is not finite.
__device__ __forceinline__ Codes m_codes(Vec<float, 8> m, float inverse, const Noise& noise) {
    m = m * inverse * 0x1p-120f;
    Codes c = {};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const unsigned u = __float_as_uint(m[k]), size = u & 0x7fffffffu;
        const unsigned code = size < 0x7f800000u ? min((size + noise.lower(k)) >> 20, 126u) : 127u;
        c.x[k / 4] |= ((u >> 24 & 128u) | code) << (8 * (k % 4));
    }
    return c;
}
__device__ __forceinline__ unsigned v_remainder(Nearest, int) { return 0x80000u; }
__device__ __forceinline__ unsigned v_remainder(const Noise& noise, int k) { return noise.upper(k); }
// The value's own exponent and upper fraction bits, after a scaling that leaves 5 bits of exponent: small
// values run into the format's subnormals as they do into those of fp32.
template <typename R> __device__ __forceinline__ Codes v_codes(Vec<float, 8> v, float inverse, const R& rounding) {
    Codes c = {};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float y = __builtin_fabsf(v[k]) * inverse * kVUnit;  // (a NaN's sign would leave no room for the remainder)
        const unsigned code = min((__float_as_uint(y) + v_remainder(rounding, k)) >> 20, 255u);  // above 255 only what is not finite
        c.x[k / 4] |= max(code, min(__float_as_uint(v[k]), 1u)) << (8 * (k % 4));   // above 0: never 0
    }
    return c;
}

__device__ __forceinline__ unsigned lane_of(unsigned x, int lane) {
    return (unsigned)__builtin_amdgcn_readlane((int)x, lane);
}

// Rounds the moments of the wave's two blocks and stores them: the codes and the blocks' scales, sm and sv being
// those of the wave's first one; `blocks` of them exist.
template <bool SPLIT, bool FULL, typename R>
__device__ __forceinline__ void store_states(const Eight<SPLIT, FULL>& e, Vec<float, 8> m, Vec<float, 8> v, unsigned char* pm,
                                             unsigned char* pv, float* sm, float* sv, int blocks, const R& rounding) {
    unsigned mt = lane_max(m), vt = lane_max(v);
    half_max(mt, vt);
    if (max(max(lane_of(mt, 31), lane_of(mt, 63)), max(lane_of(vt, 31), lane_of(vt, 63))) >= 0x7f800000u) {
        // an infinity, or a lane that has only NaN: once more without them
        mt = lane_max_finite(m);
        vt = lane_max_finite(v);
        half_max(mt, vt);
    }
    // the four quotients at once, one in each row: m and v of the first block, m and v of the second
    const int lane = threadIdx.x & 63;
    const bool of_v = lane & 16, second = lane & 32;
    const float top = __uint_as_float(second ? (of_v ? lane_of(vt, 63) : lane_of(mt, 63)) : (of_v ? lane_of(vt, 31) : lane_of(mt, 31)));
    const bool kept = top >= kTiny;
    const unsigned quotient = __float_as_uint(kept ? (of_v ? 1.0f : 448.0f) / top : 0.0f);
    const float m_inverse = __uint_as_float(second ? lane_of(quotient, 32) : lane_of(quotient, 0));
    const float v_inverse = __uint_as_float(second ? lane_of(quotient, 48) : lane_of(quotient, 16));
    const Codes mc = m_codes(m, m_inverse, rounding), all = v_codes(v, v_inverse, rounding);
    const bool v_kept = v_inverse > 0.0f;
    const Codes vc = {v_kept ? all.x[0] : 0u, v_kept ? all.x[1] : 0u};
    e.store(pm, __builtin_bit_cast(Bytes, mc));
    e.store(pv, __builtin_bit_cast(Bytes, vc));
    const int b = lane >> 5;
    if ((lane & 15) == 0 && (FULL || b < blocks))
        global(of_v ? sv : sm)[b] = kept ? (of_v ? top : top * (float)(1.0 / 448.0)) : 0.0f;
}

template <typename P, typename G, int TO, bool NOISE>
__global__ __launch_bounds__(kBlock) void adamw8_kernel(Pieces ps, GradArgs ga, AdamwArgs a) {
    const Piece c = piece_of<kWide>(ps);
    const G* g = grad_of<G>(c, ga);
    const bool skip = a.skip && *a.skip;
    if (!g || (TO != kMoves && skip)) return;
    const AdamwRates r = a.device_rates ? *a.device_rates : a.rates;
    const float f = factor_of(c, a.coefs, a.per_tensor, a.scale);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blocks = (c.n - wave * 512 + CX_STATE_BLOCK - 1) / CX_STATE_BLOCK;  // of this wave's two
    if (blocks <= 0) return;
    P* p = static_cast<P*>(c.t.param) + c.at;
    unsigned char *pm = static_cast<unsigned char*>(c.t.m) + c.at, *pv = static_cast<unsigned char*>(c.t.v) + c.at;
    float* pw = TO == kMoves ? a.moves + c.t.flat + c.at : c.t.master + c.at;
    const long long block = c.at / CX_STATE_BLOCK + wave * 2;
    float *sm = c.t.m_scale + block, *sv = c.t.v_scale + block;
    by_length<kBlock * 8>(c, [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        constexpr bool SPLIT = TO != kWeights || sizeof(P) == 4 || sizeof(G) == 4;
        const Eight<SPLIT, FULL> e(c.n);
        if constexpr (TO == kMoves)
            if (skip) return e.store(pw, Vec<float, 8>{});
        const Vec<G, 8> gx = e.load(g);
        const Codes mc = __builtin_bit_cast(Codes, e.load(pm)), vc = __builtin_bit_cast(Codes, e.load(pv));
        Vec<float, 8> w;
        if constexpr (TO == kMasters) w = e.load(pw);
        if constexpr (TO == kWeights) w = to_float<8>(e.load(p));
        const int mine = FULL || blocks > 1 ? (threadIdx.x >> 5) & 1 : 0;
        Vec<float, 8> m = m_value(mc, global(sm)[mine]), v = v_value(vc, global(sv)[mine]);
        moments<8>(to_float<8>(gx) * f, a, m, v);
        const Vec<float, 8> move = moves_of<8, false>(m, v, a, r);
        if constexpr (TO != kMoves) w = moved<8>(w, move, r.decay);
        if constexpr (TO == kMoves) e.store(pw, move);
        if constexpr (TO == kMasters) e.store(pw, w);
        if constexpr (TO != kMoves) e.store(p, from_float<P, 8>(w));
        if constexpr (NOISE) store_states(e, m, v, pm, pv, sm, sv, blocks, Noise(r.noise, c.t.flat + c.at + wave * 512));
        else store_states(e, m, v, pm, pv, sm, sv, blocks, Nearest());
    });
}

template <typename E>
__global__ __launch_bounds__(kBlock) void states_kernel(Pieces ps, E* __restrict__ m_out, E* __restrict__ v_out) {
    const Piece c = piece_of<kWide>(ps);
    const int in_piece = threadIdx.x >> 5;
    if (in_piece * CX_STATE_BLOCK >= c.n) return;
    const unsigned char *pm = static_cast<const unsigned char*>(c.t.m) + c.at, *pv = static_cast<const unsigned char*>(c.t.v) + c.at;
    const long long block = c.at / CX_STATE_BLOCK + in_piece, to = c.t.flat + c.at;
    by_length<kBlock * 8>(c, [&](auto full) {
        const Eight<sizeof(E) == 4, decltype(full)::value> e(c.n);
        const Codes mc = __builtin_bit_cast(Codes, e.load(pm)), vc = __builtin_bit_cast(Codes, e.load(pv));
        e.store(m_out + to, from_float<E, 8>(m_value(mc, global(c.t.m_scale)[block])));
        e.store(v_out + to, from_float<E, 8>(v_value(vc, global(c.t.v_scale)[block])));
    });
}

__global__ __launch_bounds__(kBlock) void set_states_kernel(Pieces ps, const float* __restrict__ m_in,
                                                            const float* __restrict__ v_in) {
    const Piece c = piece_of<kWide>(ps);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blocks = (c.n - wave * 512 + CX_STATE_BLOCK - 1) / CX_STATE_BLOCK;
    if (blocks <= 0) return;
    const long long from = c.t.flat + c.at, block = c.at / CX_STATE_BLOCK + wave * 2;
    const Eight<true, false> e(c.n);
    Vec<float, 8> v = e.load(v_in + from);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = v[k] <= 0.0f ? 0.0f : v[k];  // -0 has no code, and a square is not below it
    store_states(e, e.load(m_in + from), v, static_cast<unsigned char*>(c.t.m) + c.at,
                 static_cast<unsigned char*>(c.t.v) + c.at, c.t.m_scale + block, c.t.v_scale + block, blocks, Nearest());
}

enum Moments { k32, k8Nearest, k8Noise };

template <typename P, typename G, int TO>
void launch_step(hipStream_t s, Moments of, int n, const Pieces& ps, const GradArgs& g, const AdamwArgs& a) {
    if (of == k32) adamw32_kernel<P, G, TO><<<n, kBlock, 0, s>>>(ps, g, a);
    else if (of == k8Nearest) adamw8_kernel<P, G, TO, false><<<n, kBlock, 0, s>>>(ps, g, a);
    else adamw8_kernel<P, G, TO, true><<<n, kBlock, 0, s>>>(ps, g, a);
}

template <typename P, int TO>
void launch_step_for(int grad_type, hipStream_t s, Moments of, int n, const Pieces& ps, const GradArgs& g, const AdamwArgs& a) {
    if (grad_type == CX_F32) launch_step<P, float, TO>(s, of, n, ps, g, a);
    else if (grad_type == CX_BF16) launch_step<P, __bf16, TO>(s, of, n, ps, g, a);
    else launch_step<P, _Float16, TO>(s, of, n, ps, g, a);
}

}  // namespace

int launch_adamw(cx_handle h, cx_tensors t, const cx_grads* g, const cx_adamw_args* u, unsigned long long seed) {
    AdamwArgs a = {};
    a.beta1 = (float)u->beta1;
    a.rest1 = (float)(1.0 - u->beta1);
    a.beta2 = (float)u->beta2;
    a.rest2 = (float)(1.0 - u->beta2);
    a.eps = (float)u->eps;
    a.scale = (float)u->scale;
    a.coefs = u->n_coefs ? u->d_coefs : nullptr;
    a.per_tensor = u->n_coefs != 1;
    a.skip = u->d_skip;
    a.moves = u->d_moves;
    if (u->d_step || u->d_lr) {
        AdamwRates* rates = reinterpret_cast<AdamwRates*>(t->d_rates);
        rates_kernel<<<1, 1, 0, h->stream>>>(u->d_step, u->step, u->d_lr, u->lr, u->beta1, u->beta2, u->weight_decay,
                                             seed, u->d_skip, rates);
        CX_HIP(hipGetLastError());
        a.device_rates = rates;
    } else {
        a.rates = rates_of(u->lr, u->beta1, u->beta2, u->weight_decay, u->step, seed);
    }
    return for_grads(t, g, t->state_bits == 32 ? kFine : kWide, [&](const Pieces& ps, int n, const GradArgs& ga) -> int {
        const Moments bits = t->state_bits == 32 ? k32 : seed ? k8Noise : k8Nearest;
        hipStream_t s = h->stream;
        if (u->d_moves) launch_step_for<float, kMoves>(g->type, s, bits, n, ps, ga, a);  // (no weights: no type of theirs)
        else if (t->param_type == CX_F32) launch_step_for<float, kWeights>(g->type, s, bits, n, ps, ga, a);
        else if (t->param_type == CX_BF16 && t->masters) launch_step_for<__bf16, kMasters>(g->type, s, bits, n, ps, ga, a);
        else if (t->param_type == CX_BF16) launch_step_for<__bf16, kWeights>(g->type, s, bits, n, ps, ga, a);
        else if (t->masters) launch_step_for<_Float16, kMasters>(g->type, s, bits, n, ps, ga, a);
        else launch_step_for<_Float16, kWeights>(g->type, s, bits, n, ps, ga, a);
        CX_HIP(hipGetLastError());
        return CX_OK;
    });
}

int launch_adamw_apply(cx_handle h, cx_tensors t, const float* d_moves, float scale, double lr, const float* d_lr,
                       double weight_decay) {
    const int n = t->cut[kFine].pieces;
    if (n == 0) return CX_OK;
    const Pieces ps = t->pieces(kFine);
    const float decay = (float)(lr * weight_decay), wd = (float)weight_decay;
    hipStream_t s = h->stream;
    if (t->param_type == CX_F32) apply_kernel<float, false><<<n, kBlock, 0, s>>>(ps, d_moves, scale, decay, d_lr, wd);
    else if (t->param_type == CX_BF16 && t->masters) apply_kernel<__bf16, true><<<n, kBlock, 0, s>>>(ps, d_moves, scale, decay, d_lr, wd);
    else if (t->param_type == CX_BF16) apply_kernel<__bf16, false><<<n, kBlock, 0, s>>>(ps, d_moves, scale, decay, d_lr, wd);
    else if (t->masters) apply_kernel<_Float16, true><<<n, kBlock, 0, s>>>(ps, d_moves, scale, decay, d_lr, wd);
    else apply_kernel<_Float16, false><<<n, kBlock, 0, s>>>(ps, d_moves, scale, decay, d_lr, wd);
    CX_HIP(hipGetLastError());
    return CX_OK;
}

int launch_adamw_states(cx_handle h, cx_tensors t, int dt, void* d_m, void* d_v) {
    const int n = t->cut[kWide].pieces;
    if (n == 0) return CX_OK;
    const Pieces ps = t->pieces(kWide);
    if (dt == CX_F32) states_kernel<<<n, kBlock, 0, h->stream>>>(ps, static_cast<float*>(d_m), static_cast<float*>(d_v));
    else if (dt == CX_BF16) states_kernel<<<n, kBlock, 0, h->stream>>>(ps, static_cast<__bf16*>(d_m), static_cast<__bf16*>(d_v));
    else states_kernel<<<n, kBlock, 0, h->stream>>>(ps, static_cast<_Float16*>(d_m), static_cast<_Float16*>(d_v));
    CX_HIP(hipGetLastError());
    return CX_OK;
}

int launch_adamw_set_states(cx_handle h, cx_tensors t, const float* d_m, const float* d_v) {
    const int n = t->cut[kWide].pieces;
    if (n == 0) return CX_OK;
    set_states_kernel<<<n, kBlock, 0, h->stream>>>(t->pieces(kWide), d_m, d_v);
    CX_HIP(hipGetLastError());
    return CX_OK;
}

}  // namespace cx
